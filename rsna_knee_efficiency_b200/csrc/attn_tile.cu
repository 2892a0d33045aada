// attn_tile.cu -- attention of many query rows on the tensor cores.
//
// A piece of work = up to 256 query rows of one head of one sequence, as two tiles of 128 rows, over the key
// tiles that some row of them sees. Per key tile and query tile:
//   S = Q K^T        tcgen05 128 x 128 x D into TMEM,
//   P = 2^(S c - m)  one thread per row reads S from TMEM; P goes back to TMEM in 16 bits, over S,
//   O += P V         tcgen05 128 x D x 128, P from TMEM, V as it lies in memory.
// Two query tiles alternate: while the threads of one take the exponentials of their S, the tensor cores
// work on the other. The reference m of a row is its running maximum at the time of the last
// rescaling: O and the sum are rescaled only when the maximum has grown by more than 2^8 (then P <=
// 256, far inside fp16 and fp32), so the accumulator rarely leaves TMEM.
//
// A CTA takes one piece after the other (ask_for_block): the loads and first scores of the next piece run
// while the threads still write the last one's output.
//
// Warps 0-7 and 8-15: softmax of tile 0 and 1, two threads per row (64 scores each), then the output. Eight
// warps with 128 scores a thread took 1.3 times as long: two warps per scheduler leave it idle two cycles of
// three, waiting for their own last instruction. Warp 16: tcgen05 issue. Warp 17: TMA. Warp 18: rows of V that
// nobody may see (behind the sequence, keep = 0) are zeroed in shared memory before the product, since
// 0 * NaN is not 0 (their scores are replaced, so K may hold anything). Warp 19: which piece comes next.
#include "attn_umma.cuh"

namespace dn8 {

constexpr int AF_THREADS = 640;
// The launch gives every thread 96 registers; the softmax warps take some of the others':
// 16 x 32 x 104 + 4 x 32 x 64 = 20 x 32 x 96.
constexpr int AF_REGS_SOFTMAX = 104, AF_REGS_OTHER = 64;

template <int DP> struct TileCfg {
    static constexpr int KST = DP == 64 ? 3 : 2, VST = DP == 64 ? 3 : 2;      // stages of K and V
    static constexpr uint32_t TILE = AT_TILE * DP * 2;
    static constexpr uint32_t SMEM = 1024 + TILE * (2 + KST + VST) + 3072;
    // TMEM columns: S (and P) of the two tiles, O of the two tiles
    static constexpr uint32_t S0 = 0, O0 = 256;
};

DN8_DEV bool has_tile(const KeyTiles& k, int t) {
    return k.count > 0 && (t < k.first || (t >= k.start && t < k.start + k.count - k.first));
}
// Named barrier of two warps
DN8_DEV void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
DN8_DEV void pair_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }

struct TilePiece {
    Sequence seq;                                     // seq.b = -2: no more pieces
    int h, i0;                                        // query head, first query row
    KeyTiles all, own[2];                             // key tiles of the piece and of each query tile
    DN8_DEV bool uses(int g, int t) const { return has_tile(own[g], t); }
};

struct TileShared {
    uint64_t answer[2];                               // (16-byte aligned: first)
    uint64_t answered, qfull, qempty;
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], vok[3];
    uint64_t sfull[2], pfull[2], ofull[2], oempty[2];
    uint64_t pfilled, pread;
    TilePiece piece[2];                               // of even and odd number
    uint32_t words[3][4];
    float part[2][2][AT_TILE];                        // [tile][half of the columns][row]
    uint32_t tmem;
    int abort;
};

template <typename T, int DP>
__global__ void __launch_bounds__(AF_THREADS, 1)
attn_tile_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const dn8_attention_args a) {
    using C = TileCfg<DP>;
    static_assert(sizeof(TileShared) <= 3072, "shared state");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = smem;
    uint8_t* sk = sq + 2 * C::TILE;
    uint8_t* sv = sk + C::KST * C::TILE;
    TileShared& sh = *reinterpret_cast<TileShared*>(sv + C::VST * C::TILE);
    volatile int* abort_flag = &sh.abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 512) {
        mbar_init(&sh.answered, 1);
        mbar_init(&sh.qfull, 1);
        mbar_init(&sh.qempty, 1);
        for (int s = 0; s < 3; ++s) {
            mbar_init(&sh.kfull[s], 1);
            mbar_init(&sh.kempty[s], 1);
            mbar_init(&sh.vfull[s], 1);
            mbar_init(&sh.vempty[s], 1);
            mbar_init(&sh.vok[s], 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(&sh.sfull[g], 1);
            mbar_init(&sh.pfull[g], 8);
            mbar_init(&sh.ofull[g], 1);
            mbar_init(&sh.oempty[g], 8);
        }
        mbar_init(&sh.pfilled, 1);
        mbar_init(&sh.pread, 19);
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
        if (!mbar_wait_w(&sh.pfilled, n & 1, a.err, abort_flag, ERR_WAIT_FULL | (63 << 4))) return false;
        if (lane == 0) mbar_arrive(&sh.pread);
        return sh.piece[n & 1].seq.b >= 0;
    };

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AF_REGS_OTHER));
        if (warp == 19) {
            // ---------------- pieces ----------------
            int block = blockIdx.x, asked = 0;
            TilePiece pc;
            for (int n = 0;;) {
                pc.seq.b = -2;
                if (block >= 0) {
                    pc.seq = find_block<false>(a, block / a.Hq, 1, 2 * AT_TILE);
                    pc.h = block % a.Hq;
                }
                if (pc.seq.b >= 0) {
                    const int off = pc.seq.nk - pc.seq.nq;
                    // last blocks first: with an open left side they are the longest
                    pc.i0 = ((pc.seq.nq - 1) / (2 * AT_TILE) - pc.seq.blk) * 2 * AT_TILE;
                    const int end = min(pc.i0 + 2 * AT_TILE, pc.seq.nq);
                    pc.all = key_tiles(pc.i0 + off, end - 1 + off, pc.seq.nk, left, right, a.sinks, AT_TILE);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const int r0 = pc.i0 + g * AT_TILE;
                        pc.own[g] = key_tiles(r0 + off, min(r0 + AT_TILE, end) - 1 + off, pc.seq.nk, left, right, a.sinks,
                                              AT_TILE);
                        if (r0 >= end) pc.own[g].count = 0;
                    }
                }
                if (pc.seq.b != -1) {                 // (-1: the bound on the blocks was too high)
                    if (lane == 0) {
                        sh.piece[n & 1] = pc;
                        mbar_arrive(&sh.pfilled);
                    }
                    if (pc.seq.b == -2) break;
                    // (the softmax warps read a piece when they start on it: one is known ahead, no more)
                    if (!mbar_wait_w(&sh.pread, n & 1, a.err, abort_flag, ERR_WAIT_EMPTY | (62 << 4))) break;
                    ++n;
                }
                if (lane == 0) {
                    fence_async_smem();               // the last answer has been read
                    mbar_expect_tx(&sh.answered, 16);
                    ask_for_block(sh.answer, &sh.answered);
                }
                if (!mbar_wait_w(&sh.answered, asked & 1, a.err, abort_flag, ERR_WAIT_FULL | (61 << 4))) break;
                ++asked;
                block = answered_block(sh.answer);
                __syncwarp();
            }
        } else if (warp == 17) {
            // ---------------- TMA ----------------
            int kc = 0, vc = 0;                       // tiles loaded so far
            for (int n = 0, nq = 0; begin_piece(n); ++n) {
                const TilePiece& pc = sh.piece[n & 1];
                if (pc.all.count == 0) continue;
                if (lane == 0) {
                    const int nt = pc.i0 + AT_TILE < pc.seq.nq ? 2 : 1;
                    bool ok = mbar_wait(&sh.qempty, (nq & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (60 << 4));
                    if (ok) {
                        mbar_expect_tx(&sh.qfull, nt * C::TILE);
                        for (int g = 0; g < nt; ++g)
                            load_tile<DP>(sq + g * C::TILE, &mq, &sh.qfull, pc.h, pc.seq.q0 + pc.i0 + g * AT_TILE);
                    }
                    const int kvh = pc.h / (a.Hq / a.Hk);
                    for (int u = 0; ok && u < pc.all.count; ++u, ++kc, ++vc) {
                        const int row = pc.seq.k0 + pc.all.tile(u) * AT_TILE, ks = kc % C::KST, vs = vc % C::VST;
                        ok = mbar_wait(&sh.kempty[ks], ((kc / C::KST) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (64 << 4));
                        if (!ok) break;
                        mbar_expect_tx(&sh.kfull[ks], C::TILE);
                        load_tile<DP>(sk + ks * C::TILE, &mk, &sh.kfull[ks], kvh, row);
                        ok = mbar_wait(&sh.vempty[vs], ((vc / C::VST) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (65 << 4));
                        if (!ok) break;
                        mbar_expect_tx(&sh.vfull[vs], C::TILE);
                        load_tile<DP>(sv + vs * C::TILE, &mv, &sh.vfull[vs], kvh, row);
                    }
                }
                ++nq;
                __syncwarp();
            }
        } else if (warp == 18) {
            // ---------------- masked rows of V ----------------
            int vc = 0;
            bool ok = true;
            for (int n = 0; ok && begin_piece(n); ++n) {
                const TilePiece& pc = sh.piece[n & 1];
                for (int u = 0; u < pc.all.count; ++u, ++vc) {
                    const int t = pc.all.tile(u), vs = vc % C::VST;
                    const bool fix = a.keep != nullptr || (t + 1) * AT_TILE > pc.seq.nk;
                    uint32_t word[4];
                    if (fix)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int j = t * AT_TILE + w * 32 + lane;
                            word[w] = __ballot_sync(0xffffffffu,
                                                    j < pc.seq.nk && (a.keep == nullptr || a.keep[pc.seq.k0 + j] != 0));
                        }
                    ok = mbar_wait_w(&sh.vfull[vs], (vc / C::VST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (66 << 4));
                    if (!ok) break;
                    if (fix) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if (lane == w) sh.words[vs][w] = word[w];
                            if (!((word[w] >> lane) & 1u))
#pragma unroll
                                for (int b = 0; b < DP / 64; ++b) {
                                    uint4* row =
                                        reinterpret_cast<uint4*>(sv + vs * C::TILE + b * AT_BLOCK + (w * 32 + lane) * 128);
#pragma unroll
                                    for (int c = 0; c < 8; ++c) row[c] = make_uint4(0u, 0u, 0u, 0u);
                                }
                        }
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.vok[vs]);
                }
            }
        } else {
            // ---------------- tcgen05 issue (every value and branch uniform, see attn_umma.cuh) ----------------
            const uint32_t q0 = uniform(smem_u32(sq)), k0 = uniform(smem_u32(sk)), v0 = uniform(smem_u32(sv));
            const uint32_t tm = uniform(tmem);
            uint32_t ks = 0, kp = 0, vs = 0, vp = 0, pp = 0, qp = 0;      // stages; phases, pfull's and oempty's by bit g
            uint32_t op = 3;
            for (int n = 0; vote(begin_piece(n)); ++n) {
                KeyTiles all, own0, own1;
                {
                    const TilePiece& pc = sh.piece[n & 1];
                    all.first = uniform(pc.all.first), all.start = uniform(pc.all.start), all.count = uniform(pc.all.count);
                    own0.first = uniform(pc.own[0].first), own0.start = uniform(pc.own[0].start);
                    own0.count = uniform(pc.own[0].count);
                    own1.first = uniform(pc.own[1].first), own1.start = uniform(pc.own[1].start);
                    own1.count = uniform(pc.own[1].count);
                }
                if (vote(all.count == 0)) continue;
                if (!mbar_wait_w(&sh.qfull, qp, a.err, abort_flag, ERR_WAIT_FULL | (67 << 4))) break;
                qp ^= 1;
                bool begun0 = false, begun1 = false, had0 = false, had1 = false, ok = true;
                for (int u = 0; vote(u <= all.count); ++u) {
                    const bool more = vote(u < all.count);
                    const int t = all.tile(u);
                    const bool now0 = vote(more && has_tile(own0, t)), now1 = vote(more && has_tile(own1, t));
                    if (more) {
                        ok = mbar_wait_w(&sh.kfull[ks], kp, a.err, abort_flag, ERR_WAIT_FULL | (68 << 4));
                        if (!ok) break;
                    }
                    if (vote(u > 0)) {
                        ok = mbar_wait_w(&sh.vfull[vs], vp, a.err, abort_flag, ERR_WAIT_FULL | (69 << 4)) &&
                             mbar_wait_w(&sh.vok[vs], vp, a.err, abort_flag, ERR_WAIT_FULL | (70 << 4));
                        if (!ok) break;
                    }
                    const uint32_t kt = k0 + ks * C::TILE, vt = v0 + vs * C::TILE;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        bool& begun = g ? begun1 : begun0;
                        if (g ? had1 : had0) {
                            ok = mbar_wait_w(&sh.pfull[g], (pp >> g) & 1, a.err, abort_flag, ERR_WAIT_ACC | (71 << 4));
                            if (!ok) break;
                            pp ^= 1u << g;
                            if (!begun) {             // the last piece's output has been read
                                ok = mbar_wait_w(&sh.oempty[g], (op >> g) & 1, a.err, abort_flag, ERR_WAIT_ACC | (59 << 4));
                                if (!ok) break;
                                op ^= 1u << g;
                            }
                            tc_fence_after();
                            mma_values<T, DP, 64>(tm + C::O0 + g * DP, tm + C::S0 + g * 128, vt, begun);
                            begun = true;
                        }
                        if (g ? now1 : now0) {
                            // (S lies over P: the product that reads P was issued before)
                            tc_fence_after();
                            mma_scores<T, DP>(tm + C::S0 + g * 128, q0 + g * C::TILE, kt);
                            umma_commit_w(&sh.sfull[g]);
                        }
                    }
                    if (!ok) break;
                    had0 = now0;
                    had1 = now1;
                    if (more) {
                        umma_commit_w(&sh.kempty[ks]);
                        if (++ks == C::KST) {
                            ks = 0;
                            kp ^= 1;
                        }
                    }
                    if (vote(u + 1 == all.count)) umma_commit_w(&sh.qempty);
                    if (vote(u > 0)) {
                        umma_commit_w(&sh.vempty[vs]);
                        if (++vs == C::VST) {
                            vs = 0;
                            vp ^= 1;
                        }
                    }
                }
                if (!ok) break;
                if (begun0) umma_commit_w(&sh.ofull[0]);
                if (begun1) umma_commit_w(&sh.ofull[1]);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AF_REGS_SOFTMAX));
        // ---------------- softmax: two threads per row ----------------
        const int g = warp >> 3, half = (warp >> 2) & 1, row = (warp & 3) * 32 + lane;
        const uint32_t quad = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::S0 + g * 128 + half * 64 + quad, to = tmem + C::O0 + g * DP + half * (DP / 2) + quad;
        float* mine = &sh.part[g][half][row];
        const float* other = &sh.part[g][half ^ 1][row];
        const int pair = 1 + g * 4 + (warp & 3);      // named barrier of the two warps that share rows
        const float sc = a.scale * ATT_LOG2E;
        int ns = 0, no = 0, vc0 = 0;                  // scores and outputs so far; V tiles before this piece
        bool ok = true;
        for (int np = 0; ok && begin_piece(np); ++np) {
            const TilePiece& pc = sh.piece[np & 1];
            float m = -INFINITY, l = 0.0f;            // reference (times sc), and this half's sum
            int n = 0;
            for (int u = 0; u < pc.all.count; ++u) {
                const int t = pc.all.tile(u), j0 = t * AT_TILE, vs = (vc0 + u) % C::VST;
                if (!pc.uses(g, t)) continue;
                // positions of the tile's first and last row: does every row see every key?
                const int nk = pc.seq.nk, last = j0 + AT_TILE - 1, pa = pc.i0 + g * AT_TILE + nk - pc.seq.nq;
                const bool masked = a.keep != nullptr || last > min(nk - 1, pa + right) ||
                                    (j0 < min(pa + AT_TILE, nk) - 1 - left && last >= a.sinks);
                uint32_t word[2];
                if (masked) {
                    const int hi = min(nk - 1, pa + row + right) - j0, lo = pa + row - left - j0;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        word[c] = bits_upto(hi, 2 * half + c) &
                                  (bits_from(lo, 2 * half + c) | bits_upto(a.sinks - 1 - j0, 2 * half + c));
                }
                ok = mbar_wait_w(&sh.sfull[g], ns & 1, a.err, abort_flag, ERR_WAIT_ACC | (73 << 4));
                if (!ok) break;
                ++ns;
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(ts, r[0]);
                tmem_ld32(ts + 32, r[1]);
                if (a.keep != nullptr) {
                    // (after S: its issue has waited for the V tiles before this one, so the phase is not mistaken)
                    ok = mbar_wait_w(&sh.vok[vs], ((vc0 + u) / C::VST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (72 << 4));
#pragma unroll
                    for (int c = 0; c < 2; ++c) word[c] &= sh.words[vs][2 * half + c];
                }
                tmem_wait_ld(r[0]);
                reg_bind(r[1]);
                if (!ok) break;
                if (masked)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e) r[c][e] = (word[c] >> e) & 1u ? r[c][e] : 0xFF800000u;   // -inf
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // four chains, not one of 64
#pragma unroll
                for (int e = 0; e < 32; e += 4)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        m4[c] = fmaxf(fmaxf(m4[c], __uint_as_float(r[c >> 1][e + 2 * (c & 1)])),
                                      __uint_as_float(r[c >> 1][e + 2 * (c & 1) + 1]));
                float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                *mine = mx;
                pair_sync(pair);
                if (*abort_flag) {
                    ok = false;
                    break;
                }
                mx = fmaxf(mx, *other) * sc;
                if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                    const float mn = fmaxf(m, mx);
                    const float f = ex2(m - (mn == -INFINITY ? 0.0f : mn));
                    m = mn;
                    l *= f;
                    if (n > 0) {
                        // S complete: so is the product before it, and the next one waits for P
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t o[16];
                            tmem_ld16(to + 16 * c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(to + 16 * c, o);
                            tmem_wait_st(o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                const float2 sc2 = f2_pack(sc, sc), mr2 = f2_pack(-ref, -ref);
                float2 s2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
                uint32_t pk[2][16];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 x = f2_fma(f2_pack(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), sc2, mr2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        s2[e & 1] = __fadd2_rn(s2[e & 1], x);
                        // the weights are rounded to the values' type, the type of the matrix instruction
                        pk[c][e] = pack2(T(), x.x, x.y);
                    }
                    tmem_st16(ts + 16 * c, pk[c]);
                }
                l += (s2[0].x + s2[0].y) + (s2[1].x + s2[1].y);
                tmem_wait_st(pk[0]);
                tmem_wait_st(pk[1]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.pfull[g]);
                ++n;
            }
            if (!ok) break;
            vc0 += pc.all.count;
            if (n > 0) {
                // the two halves' sums (the barrier before has been passed by both: part is free)
                pair_sync(pair);
                *mine = l;
                pair_sync(pair);
                l = half == 0 ? l + *other : *other + l;
                pair_sync(pair);
                ok = mbar_wait_w(&sh.ofull[g], no & 1, a.err, abort_flag, ERR_WAIT_ACC | (74 << 4));
                if (!ok || *abort_flag) break;
                ++no;
                tc_fence_after();
            }
            const int i = pc.i0 + g * AT_TILE + row, h = pc.h;
            const int64_t at = pc.seq.q0 + i;
            const bool live = i < pc.seq.nq;
            T* out = static_cast<T*>(a.out) + at * a.o_stride_t + static_cast<int64_t>(h) * a.o_stride_h;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[16] = {};
                if (n > 0) {
                    tmem_ld16(to + 16 * c, o);
                    tmem_wait_ld(o);
                }
                const int d = half * (DP / 2) + 16 * c;
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = l > 0.0f ? __uint_as_float(o[e + x]) * inv : 0.0f;
                    if (live && d + e < a.D) store_f32(out + d + e, v);
                }
            }
            if (n > 0) {                              // O has been read: the next piece may use it
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.oempty[g]);
            }
            if (live && half == 0 && a.lse != nullptr)
                a.lse[at * a.Hq + h] = l > 0.0f ? (m + __log2f(l)) * ATT_LN2 : -INFINITY;
        }
        // A warp that gave up arrives once more, so that its partner's barrier completes; the partner then
        // sees the abort flag and leaves too.
        if (*abort_flag) pair_arrive(pair);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t make_head_map(CUtensorMap* map, const void* base, int type, int64_t rows, int heads, int D, int64_t stride_t,
                          int64_t stride_h, int box_rows) {
    static EncodeTiledFn encode = nullptr;
    if (encode == nullptr) {
        cudaDriverEntryPointQueryResult q;
        void* fn = nullptr;
        cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || fn == nullptr) return cudaErrorNotSupported;
        encode = reinterpret_cast<EncodeTiledFn>(fn);
    }
    // (an extent of one needs no stride: any valid one will do)
    if (heads == 1) stride_h = D;
    if (rows == 1) stride_t = stride_h * heads;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride_h) * 2, static_cast<cuuint64_t>(stride_t) * 2};
    cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(box_rows)};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType t = type == DN8_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUresult r = encode(map, t, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int DP> static cudaError_t tile_go(const dn8_attention_args& a, cudaStream_t st) {
    CUtensorMap mq = {}, mk = {}, mv = {};
    cudaError_t e = make_head_map(&mq, a.q, a.type, a.Tq, a.Hq, a.D, a.q_stride_t, a.q_stride_h);
    if (e == cudaSuccess && a.Tk > 0) e = make_head_map(&mk, a.k, a.type, a.Tk, a.Hk, a.D, a.k_stride_t, a.k_stride_h);
    if (e == cudaSuccess && a.Tk > 0) e = make_head_map(&mv, a.v, a.type, a.Tk, a.Hk, a.D, a.v_stride_t, a.v_stride_h);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(attn_tile_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    // a bound on the blocks: every sequence may leave one unfilled
    const int64_t blocks = (a.Tq / (2 * AT_TILE) + (a.B < a.Tq ? a.B : a.Tq)) * a.Hq;
    if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    return launch_pdl(false, attn_tile_kernel<T, DP>, dim3(static_cast<unsigned>(blocks)), dim3(AF_THREADS),
                      TileCfg<DP>::SMEM, st, mq, mk, mv, a);
}

cudaError_t launch_attention_tile(const dn8_attention_args& a, cudaStream_t st) {
    if (a.type == DN8_F16) return a.D <= 64 ? tile_go<__half, 64>(a, st) : tile_go<__half, 128>(a, st);
    return a.D <= 64 ? tile_go<__nv_bfloat16, 64>(a, st) : tile_go<__nv_bfloat16, 128>(a, st);
}

}  // namespace dn8
