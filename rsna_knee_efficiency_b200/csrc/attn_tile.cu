// attn_tile.cu -- attention of many query rows on the tensor cores.
//
// A piece of work = up to 256 query rows of one head of one sequence, as two tiles of 128 rows, over the key
// tiles that some row of them sees. Per key tile and query tile:
//   S = Q K^T        tcgen05 128 x 128 x D into TMEM,
//   P = 2^(S c - m)  the threads read S from TMEM; P goes back to TMEM in 16 bits,
//   O += P V         tcgen05 128 x D x 128, P from TMEM, V as it lies in memory.
// Two query tiles are worked on side by side. At D <= 64 P has TMEM columns of its own, so the next S is made as
// soon as this one has been read, and the threads find it when they are done; above, P lies over S, and the
// next S waits for the product that reads P. The reference m of a row is its running maximum at the time of the last
// rescaling: O and the sum are rescaled only when the maximum has grown by more than 2^8 (then P <=
// 256, far inside fp16 and fp32), so the accumulator rarely leaves TMEM.
//
// A CTA takes one piece after the other (ask_for_block): the loads and first scores of the next piece run
// while the threads still write the last one's output. A piece costs some 5 us beyond its tiles (1.4 us each at
// D <= 64), so for short sequences the next one is asked for early and looked up in shared memory: 128 x 128
// tokens, 16 heads, D = 64, 66 us (with the question behind V and offsets from memory it was 90, not 74).
//
// In bursts at 1965 MHz: 2 x 8192 tokens, 16 heads, no mask, D = 64 689 us (798 TFLOP/s; the exponentials alone take
// 0.67 of it at the special function units' rate), D = 128 1006 us (1093 TFLOP/s, 0.64 of the measured matrix rate).
// Four views of 6144, causal, 8 heads, D = 128: 340 us, and 370 in a loop, where the power cap holds the clock at
// 1715 MHz. Bound by the latency of a tile's steps: issue slots, special function units and tensor cores are each
// busy for 0.41 to 0.56, 0.48 and 0.24 to 0.48 of the time (windows at D = 64, causal at D = 128).
//
// Warps 0-7 and 8-15: softmax of tile 0 and 1, a warp per 16 rows and four threads per row, so that a row's
// maximum takes two shuffles (32 scores of two rows a thread; one thread per row left the schedulers idle
// two cycles of three, two threads of different warps per row had to meet in shared memory for every
// tile). Warps 16 and 19: tcgen05 issue, one per query tile: an issue is some 25 instructions with its waits,
// and one warp for both tiles was late for each by the other's. Warp 17: TMA. Warp 18: which piece comes
// next, and rows of V that nobody may see (behind the sequence, keep = 0, before every window): they are zeroed in
// shared memory before the product, since 0 * NaN is not 0 (their scores are replaced, so K may hold anything).
#include "attn_umma.cuh"

namespace dn8 {

constexpr int AF_THREADS = 640;
// The launch gives every thread 96 registers; the softmax warps take some of the others':
// 16 x 32 x 104 + 4 x 32 x 64 = 20 x 32 x 96.
constexpr int AF_REGS_SOFTMAX = 104, AF_REGS_OTHER = 64;
// How many tiles before the end of a piece the next one is asked for: time enough to hide the question and the
// first loads. Asked for at the start, a piece waits behind a long one while others run out of work: four
// sequences of 6144, causal, D = 128, take 360 us instead of 344 (in a loop under the power cap 383, not 371).
constexpr int AF_AHEAD = 4;
constexpr float AF_SHARE = 4.0f;                      // key tiles of a share, at least

template <int DP> struct TileCfg {
    static constexpr int KST = DP == 64 ? 3 : 2, VST = DP == 64 ? 3 : 2;      // stages of K and V
    static constexpr uint32_t TILE = AT_TILE * DP * 2;
    static constexpr uint32_t SMEM = 1024 + TILE * (2 + KST + VST) + 8192;
    // TMEM columns: S of the two tiles, P (over S, or of its own), O
    static constexpr bool OWN_P = DP == 64;
    static constexpr uint32_t S0 = 0, P0 = OWN_P ? 256 : 0, PG = OWN_P ? 64 : 128, O0 = OWN_P ? 384 : 256;
};

// Named barrier of the two warps that share 32 TMEM lanes
DN8_DEV void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
DN8_DEV void pair_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }

struct TilePiece {
    Sequence seq;                                     // seq.b = -2: no more pieces
    int h, i0;                                        // query head, first query row
    int share;                                        // where a share's results go, or -1: straight to the output
    KeyTiles all, own[2];                             // key tiles of the piece, and of each query tile
    // Query tile g's own are the piece's tiles u < lead[g] and from[g] <= u < to[g]. A tile whose first key is above
    // hic[g], or below loc[g] but above skc, or (with a key mask) every tile, needs a mask.
    int lead[2], from[2], to[2], hic[2], loc[2], skc;
};

// Shares of a piece's key tiles. Where the rows make fewer pieces than half the SMs (a few heads, or some hundreds
// of queries over long caches), a piece whose walk is longer than an SM's part of all of them is cut. The
// lengths are known to the GPU alone, so each CTA adds them up: pieces times the tiles that a piece sees at
// most. A piece gets as many shares as whole parts fit into its sequence's, so all shares run side by side.
// Uncut and cut, us: one head, 5627 queries and keys, D = 80, 178 and 60; two heads, 1905, D = 128, window of
// 1450, 51 and 42; four heads, 4096, D = 64, 66 and 56; 64 queries of 4 heads over 20000 keys 113 and 30. A call whose
// pieces turn out not to be cut pays 8 us for this and the join (12 heads, 4096: 105 and 114).
struct TilePlan {
    int sms;                                          // 0: nothing is cut
    int units;                                        // pieces and shares, per head (a bound)
    float* o;                                         // [share][256][DP], relative to the reference
    float2* ml;                                       // [share][256] (reference, sum)
    int4* rec;                                        // [share] first row, rows (0: not a piece's first share), shares
};
struct TileShares {
    const dn8_attention_args& a;
    float inv;                                        // 1 / tiles of a part, or 0: nothing is cut
    DN8_DEV int tiles(int nq, int nk) const { return (seen_keys(a, min(nq, 2 * AT_TILE), nk) + AT_TILE - 1) / AT_TILE; }
    DN8_DEV int operator()(int nq, int nk) const { return max(1, static_cast<int>(tiles(nq, nk) * inv)); }
};
DN8_DEV TileShares tile_shares(const dn8_attention_args& a, const TilePlan& plan) {      // (one whole warp)
    TileShares s = {a, 0.0f};
    float total = 0.0f;
    for (int b = threadIdx.x & 31; b < a.B; b += 32) {
        const Sequence q = sequence_of(a, b);
        total += static_cast<float>((q.nq + 2 * AT_TILE - 1) / (2 * AT_TILE)) * static_cast<float>(s.tiles(q.nq, q.nk));
    }
    s.inv = fminf(static_cast<float>(plan.sms) / (warp_sum(total) * static_cast<float>(a.Hq)), 1.0f / AF_SHARE);
    return s;
}

struct TileShared {
    uint64_t answer[2];                               // (16-byte aligned: first)
    uint64_t answered, qfull, qempty;
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], vok[3];
    uint64_t sfull[2], sread[2], pfull[2], ofull[2], oempty[2];
    uint64_t pfilled, pread;
    TilePiece piece[2];                               // of even and odd number
    uint32_t words[3][4];
    float stat[2][2][2][AT_TILE];                     // [turn][tile][sum, reference][row]
    SequenceTable table;
    uint32_t tmem;
    int abort;
};

template <typename T, int DP, bool CUT>
__global__ void __launch_bounds__(AF_THREADS, 1)
attn_tile_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const dn8_attention_args a, const TilePlan plan) {
    using C = TileCfg<DP>;
    static_assert(sizeof(TileShared) <= 8192, "shared state");
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
        mbar_init(&sh.qempty, 2);
        for (int s = 0; s < 3; ++s) {
            mbar_init(&sh.kfull[s], 1);
            mbar_init(&sh.kempty[s], 2);
            mbar_init(&sh.vfull[s], 1);
            mbar_init(&sh.vempty[s], 2);
            mbar_init(&sh.vok[s], 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(&sh.sfull[g], 1);
            mbar_init(&sh.sread[g], 8);
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
    // next one. Every warp but 18 calls this for n = 0, 1, ... when it begins; false: there is
    // none (or a wait gave up).
    auto begin_piece = [&](int n) -> bool {
        if (!mbar_wait_w(&sh.pfilled, n & 1, a.err, abort_flag, ERR_WAIT_FULL | (63 << 4))) return false;
        if (lane == 0) mbar_arrive(&sh.pread);
        return sh.piece[n & 1].seq.b >= 0;
    };

    if (CUT) griddep_launch_dependents();
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AF_REGS_OTHER));
        if (warp == 18) {
            // ---------------- pieces, and masked rows of V ----------------
            int block = blockIdx.x, asked = 0, vc = 0;
            const TileShares shares = CUT ? tile_shares(a, plan) : TileShares{a, 0.0f};
            const bool few = a.B <= SequenceTable::MOST;
            if (few) sh.table.fill<false>(a, 2 * AT_TILE, shares);
            TilePiece pc;
            // Looks block after block up until one holds a piece: false after the last.
            auto look = [&]() -> bool {
                while (block >= 0) {
                    pc.seq = few ? sh.table.find(a.B, block / a.Hq) : find_block<false>(a, block / a.Hq, 1, 2 * AT_TILE, shares);
                    if (CUT) {
                        pc.share = block;
                        // (behind the last piece there are some 148 blocks with nothing to do: one of them ends this CTA's
                        // search, blocks that were not asked for start by themselves. Each one more held V up for
                        // 2 us.)
                        if (pc.seq.b < 0) {
                            if (lane == 0) plan.rec[block] = make_int4(0, 0, 0, 0);
                            return false;
                        }
                    }
                    pc.h = block % a.Hq;
                    if (pc.seq.b >= 0) return true;   // (the bound on the blocks may be too high)
                    if (lane == 0) {
                        fence_async_smem();           // the last answer has been read
                        mbar_expect_tx(&sh.answered, 16);
                        ask_for_block(sh.answer, &sh.answered);
                    }
                    if (!mbar_wait_w(&sh.answered, asked & 1, a.err, abort_flag, ERR_WAIT_FULL | (61 << 4))) return false;
                    ++asked;
                    block = answered_block(sh.answer);
                    __syncwarp();
                }
                return false;
            };
            auto publish = [&](int n, bool there) {
                if (!there) {
                    pc.seq.b = -2;
                } else {
                    const int nq = pc.seq.nq, nk = pc.seq.nk, off = nk - nq;
                    const int cuts = CUT ? shares(nq, nk) : 1, nth = cuts == 1 ? pc.seq.blk : pc.seq.blk / cuts;
                    const int mine = pc.seq.blk - nth * cuts;
                    // last blocks first: with an open left side they are the longest
                    pc.i0 = ((nq - 1) / (2 * AT_TILE) - nth) * 2 * AT_TILE;
                    const int end = min(pc.i0 + 2 * AT_TILE, nq);
                    const KeyTiles whole = key_tiles(pc.i0 + off, end - 1 + off, nk, left, right, a.sinks, AT_TILE);
                    pc.all = whole;
                    int u0 = 0, n_ = whole.count;     // this share's of the piece's tiles: n_ from u0 on
                    if (CUT) {
                        const bool first = cuts > 1 && mine == 0;
                        if (lane == 0) plan.rec[pc.share] = make_int4(pc.seq.q0 + pc.i0, first ? end - pc.i0 : 0, cuts, 0);
                        if (cuts > 1) {
                            // (tiles < 2^21, and at most one share per SM)
                            u0 = mine * whole.count / cuts;
                            n_ = (mine + 1) * whole.count / cuts - u0;
                            pc.all.cut(u0, u0 + n_);
                        } else {
                            pc.share = -1;
                        }
                    }
                    pc.skc = a.sinks - AT_TILE;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const int p0 = pc.i0 + g * AT_TILE + off, p1 = min(pc.i0 + (g + 1) * AT_TILE, end) - 1 + off;
                        KeyTiles own = key_tiles(p0, p1, nk, left, right, a.sinks, AT_TILE);
                        if (p0 > p1) own.first = own.count = 0;
                        // (a query tile's own are among the piece's)
                        const int from = own.count > 0 ? whole.first + own.start - whole.start : 0;
                        pc.lead[g] = max(0, min(own.first - u0, n_));
                        pc.from[g] = max(0, min(from - u0, n_));
                        pc.to[g] = max(0, min(from + own.count - own.first - u0, n_));
                        pc.own[g].base = pc.all.base;
                        pc.own[g].first = pc.lead[g];
                        pc.own[g].start = pc.all.tile(pc.from[g]);
                        pc.own[g].count = pc.lead[g] + max(0, pc.to[g] - pc.from[g]);
                        pc.hic[g] = min(nk - 1, p0 + right) - (AT_TILE - 1);
                        pc.loc[g] = p1 - left;
                    }
                }
                if (lane == 0) {
                    sh.piece[n & 1] = pc;
                    mbar_arrive(&sh.pfilled);
                }
                __syncwarp();
            };
            pc.share = -1;
            publish(0, look());
            bool ok = true;
            for (int n = 0; pc.seq.b >= 0; ++n) {
                const int count = pc.all.count, nk = pc.seq.nk, k0 = pc.seq.k0;
                const KeyTiles all = pc.all;
                const uint32_t hidden = hidden_keys(a, pc.seq.nq, nk);
                const int ask_at = max(0, count - AF_AHEAD);
                for (int u = 0; u < max(count, 1); ++u) {
                    if (u == ask_at) {
                        // The next piece, asked for once every warp has begun with this one ...
                        ok = mbar_wait_w(&sh.pread, n & 1, a.err, abort_flag, ERR_WAIT_EMPTY | (62 << 4));
                        if (!ok) break;
                        if (lane == 0) {
                            fence_async_smem();
                            mbar_expect_tx(&sh.answered, 16);
                            ask_for_block(sh.answer, &sh.answered);
                        }
                    }
                    if (u < count) {
                        const int t = all.tile(u), vs = vc % C::VST;
                        const bool fix = a.keep != nullptr || (t + 1) * AT_TILE > nk ||
                                         (hidden > 0 && t * AT_TILE < a.sinks + static_cast<int>(hidden) &&
                                          (t + 1) * AT_TILE > a.sinks);
                        uint32_t word[4];
                        if (fix)
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const int j = t * AT_TILE + w * 32 + lane;
                                word[w] = __ballot_sync(0xffffffffu, j < nk && behind_hidden(a, j, hidden) &&
                                                                         (a.keep == nullptr || a.keep[k0 + j] != 0));
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
                        ++vc;
                    }
                    if (u == ask_at) {
                        // ... and looked up when this tile's V, whose product may be waiting, has been let go
                        ok = mbar_wait_w(&sh.answered, asked & 1, a.err, abort_flag, ERR_WAIT_FULL | (61 << 4));
                        if (!ok) break;
                        ++asked;
                        block = answered_block(sh.answer);
                        __syncwarp();
                        const bool there = look();
                        publish(n + 1, there);
                    }
                }
                if (!ok) break;
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
        } else {
            // ---------------- tcgen05 issue (every value and branch uniform, see attn_umma.cuh) ----------------
            // warp 16: query tile 0, warp 19: query tile 1
            const uint32_t g = vote(warp == 19) ? 1u : 0u;
            const uint32_t q0 = uniform(smem_u32(sq) + g * C::TILE), k0 = uniform(smem_u32(sk)), v0 = uniform(smem_u32(sv));
            const uint32_t ts = uniform(tmem + C::S0 + g * 128), tp = uniform(tmem + C::P0 + g * C::PG);
            const uint32_t to = uniform(tmem + C::O0 + g * DP);
            uint32_t ks = 0, kp = 0, vs = 0, vp = 0, pp = 0, qp = 0, op = 1, rp = 1;      // stages and phases
            for (int n = 0; vote(begin_piece(n)); ++n) {
                const TilePiece& pc = sh.piece[n & 1];
                const int count = uniform(pc.all.count), lead = uniform(pc.lead[g]), from = uniform(pc.from[g]),
                          to_ = uniform(pc.to[g]);
                if (vote(count == 0)) continue;
                bool ok = mbar_wait_w(&sh.qfull, qp, a.err, abort_flag, ERR_WAIT_FULL | (67 << 4)), begun = false, had = false;
                if (!ok) break;
                qp ^= 1;
                // The next scores: of key tile u, and its release. (A tile that this query tile does not use is waited
                // for all the same before it is released: the release counts for the phase that follows its load.)
                auto scores = [&](int u, bool now) {
                    if (now) {
                        // (S is free: read, or P over it multiplied)
                        if (C::OWN_P) {
                            ok = mbar_wait_w(&sh.sread[g], rp, a.err, abort_flag, ERR_WAIT_ACC | (55 << 4));
                            if (!ok) return;
                            rp ^= 1;
                        }
                        tc_fence_after();
                        mma_scores<T, DP>(ts, q0, k0 + ks * C::TILE);
                        umma_commit_w(&sh.sfull[g]);
                    }
                    umma_commit_w(&sh.kempty[ks]);
                    if (++ks == C::KST) {
                        ks = 0;
                        kp ^= 1;
                    }
                    if (vote(u + 1 == count)) umma_commit_w(&sh.qempty);
                };
                for (int u = 0; vote(u <= count); ++u) {
                    const bool more = vote(u < count), now = vote(more && (u < lead || (u >= from && u < to_)));
                    if (more) {
                        ok = mbar_wait_w(&sh.kfull[ks], kp, a.err, abort_flag, ERR_WAIT_FULL | (68 << 4));
                        if (!ok) break;
                        if (C::OWN_P) scores(u, now);
                        if (!ok) break;
                    }
                    if (vote(u > 0)) {
                        ok = mbar_wait_w(&sh.vok[vs], vp, a.err, abort_flag, ERR_WAIT_FULL | (70 << 4));
                        if (!ok) break;
                        if (had) {
                            ok = mbar_wait_w(&sh.pfull[g], pp, a.err, abort_flag, ERR_WAIT_ACC | (71 << 4));
                            if (!ok) break;
                            pp ^= 1;
                            if (!begun) {             // the last piece's output has been read
                                ok = mbar_wait_w(&sh.oempty[g], op, a.err, abort_flag, ERR_WAIT_ACC | (59 << 4));
                                if (!ok) break;
                                op ^= 1;
                            }
                            tc_fence_after();
                            mma_values<T, DP, 128>(to, tp, v0 + vs * C::TILE, begun);
                            if (C::OWN_P) umma_commit_w(&sh.ofull[g]);
                            begun = true;
                        }
                    }
                    if (!C::OWN_P && more) scores(u, now);
                    if (vote(u > 0)) {
                        umma_commit_w(&sh.vempty[vs]);
                        if (++vs == C::VST) {
                            vs = 0;
                            vp ^= 1;
                        }
                    }
                    had = now;
                }
                if (!ok) break;
                if (!C::OWN_P && begun) umma_commit_w(&sh.ofull[g]);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AF_REGS_SOFTMAX));
        // ---------------- softmax: a warp per 16 rows, four threads per row ----------------
        const int g = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
        const int row = quad * 32 + half * 16 + (lane >> 2);           // of the query tile; the other one is row + 8
        const uint32_t lanes = static_cast<uint32_t>(quad * 32 + half * 16) << 16;
        const uint32_t ts = tmem + C::S0 + g * 128 + lanes, tp = tmem + C::P0 + g * C::PG + lanes, to = tmem + C::O0 + g * DP + lanes;
        const int pair = 1 + g * 4 + quad;
        const float sc = a.scale * ATT_LOG2E;
        int ns = 0, no = 0, vc0 = 0;                  // scores and outputs so far; V tiles before this piece
        int hand = 0;                                // outputs handed over so far, odd or even
        bool ok = true;
        for (int np = 0; ok && begin_piece(np); ++np) {
            const TilePiece& pc = sh.piece[np & 1];
            const int tiles = pc.own[g].count, turn = pc.own[g].base + pc.own[g].first - 1, hic = pc.hic[g], loc = pc.loc[g], skc = pc.skc;
            int t = pc.own[g].tile(0);
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};      // references (times sc), this thread's sums
            for (int n = 0; n < tiles; ++n) {
                const int j0 = t * AT_TILE;
                const bool ranged = j0 > hic || (j0 < loc && j0 > skc), masked = a.keep != nullptr || ranged;
                t = t == turn ? pc.own[g].start : t + 1;
                ok = mbar_wait_w(&sh.sfull[g], ns & 1, a.err, abort_flag, ERR_WAIT_ACC | (73 << 4));
                if (!ok) break;
                ++ns;
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld16x256_8(ts, r[0]);
                tmem_ld16x256_8(ts + 64, r[1]);
                if (masked) {
                    uint32_t keep[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (a.keep != nullptr) {
                        // (after S: its issue has waited for the V tiles VST before, so the phase is not mistaken)
                        const int u = vc0 + (n < pc.lead[g] ? n : pc.from[g] + n - pc.lead[g]), vs = u % C::VST;
                        ok = mbar_wait_w(&sh.vok[vs], (u / C::VST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (72 << 4));
#pragma unroll
                        for (int w = 0; w < 4; ++w) keep[w] = sh.words[vs][w];
                    }
                    tmem_wait_ld(r[0]);
                    reg_bind(r[1]);
                    if (!ok) break;
                    const int nk = pc.seq.nk, p0 = pc.i0 + g * AT_TILE + row + nk - pc.seq.nq;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t word = keep[w];
                            if (ranged) {
                                const int p = p0 + 8 * h, hi = min(nk - 1, p + right) - j0, lo = p - left - j0;
                                word &= bits_upto(hi, w) & (bits_from(lo, w) | bits_upto(a.sinks - 1 - j0, w));
                            }
                            word >>= 2 * (lane & 3);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    uint32_t& x = r[w >> 1][4 * (4 * (w & 1) + k) + 2 * h + e];
                                    x = (word >> (8 * k + e)) & 1u ? x : 0xFF800000u;          // -inf
                                }
                        }
                } else {
                    tmem_wait_ld(r[0]);
                    reg_bind(r[1]);
                }
                if (C::OWN_P) {                       // S is in registers: the next one may come
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.sread[g]);
                }
                float mx[2][2] = {{-INFINITY, -INFINITY}, {-INFINITY, -INFINITY}};
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            mx[h][c] = fmaxf(fmaxf(mx[h][c], __uint_as_float(r[c][4 * k + 2 * h])),
                                             __uint_as_float(r[c][4 * k + 2 * h + 1]));
                float top[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(mx[h][0], mx[h][1]);
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2)) * sc;
                }
                if (C::OWN_P && n > 0) {              // the product before is done with P, and O may be rescaled
                    ok = mbar_wait_w(&sh.ofull[g], no & 1, a.err, abort_flag, ERR_WAIT_ACC | (56 << 4));
                    if (!ok) break;
                    ++no;
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
                    float f[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float mn = fmaxf(m[h], top[h]);
                        f[h] = ex2(m[h] - (mn == -INFINITY ? 0.0f : mn));
                        m[h] = mn;
                        l[h] *= f[h];
                    }
                    if (n > 0) {
                        // (with P over S: S complete, so is the product before it; the next one waits for P)
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t o[16];
                            tmem_ld16x256_4(to + 32 * c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f[(e >> 1) & 1]);
                            tmem_st16x256_4(to + 32 * c, o);
                            tmem_wait_st(o);
                        }
                    }
                }
                const float2 sc2 = f2_pack(sc, sc);
                float2 mr2[2], s2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float ref = m[h] == -INFINITY ? 0.0f : -m[h];
                    mr2[h] = f2_pack(ref, ref);
                }
                uint32_t pk[2][16];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 x = f2_fma(f2_pack(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), sc2,
                                          mr2[e & 1]);
                        // (some of them by polynomial, to spare the special function units, cost the schedulers as
                        // much as it spared)
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        s2[e & 1] = __fadd2_rn(s2[e & 1], x);
                        // the weights are rounded to the values' type, the type of the matrix instruction
                        pk[c][e] = pack2(T(), x.x, x.y);
                    }
                    tmem_st16x128_8(tp + 32 * c, pk[c]);
                }
                l[0] += s2[0].x + s2[0].y;
                l[1] += s2[1].x + s2[1].y;
                tmem_wait_st(pk[0]);
                tmem_wait_st(pk[1]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.pfull[g]);
            }
            if (!ok) break;
            vc0 += pc.all.count;
            // The output: a row per thread, the two warps of these 32 rows half of the elements each. Sums and
            // references change hands through shared memory, by turns in two places: a warp writes to a place again
            // only after the barrier of the turn between, which its partner reaches when it has read this one. (Key
            // tiles do not keep the two together: a piece of one tile waits for nobody before its sums are written.)
            float ls = 0.0f, ms = -INFINITY;
            if (tiles > 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                    if ((lane & 3) == 0) {
                        sh.stat[hand][g][0][row + 8 * h] = l[h];
                        sh.stat[hand][g][1][row + 8 * h] = m[h];
                    }
                }
                pair_sync(pair);
                ls = sh.stat[hand][g][0][quad * 32 + lane];
                ms = sh.stat[hand][g][1][quad * 32 + lane];
                hand ^= 1;
                ok = mbar_wait_w(&sh.ofull[g], no & 1, a.err, abort_flag, ERR_WAIT_ACC | (74 << 4));
                if (!ok || *abort_flag) break;
                ++no;
                tc_fence_after();
            }
            const int i = pc.i0 + g * AT_TILE + quad * 32 + lane, h = pc.h;
            const int64_t at = pc.seq.q0 + i;
            const bool live = i < pc.seq.nq;
            T* out = static_cast<T*>(a.out) + at * a.o_stride_t + static_cast<int64_t>(h) * a.o_stride_h;
            const uint32_t tq = tmem + C::O0 + g * DP + half * (DP / 2) + (static_cast<uint32_t>(quad * 32) << 16);
            const float inv = ls > 0.0f ? 1.0f / ls : 0.0f;
            const bool cut = CUT && pc.share >= 0;
            const int64_t slot = static_cast<int64_t>(pc.share) * 2 * AT_TILE + g * AT_TILE + quad * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[16] = {};
                if (tiles > 0) {
                    tmem_ld16(tq + 16 * c, o);
                    tmem_wait_ld(o);
                }
                const int d = half * (DP / 2) + 16 * c;
                if (cut) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        if (live) *reinterpret_cast<uint4*>(plan.o + slot * DP + d + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = ls > 0.0f ? __uint_as_float(o[e + x]) * inv : 0.0f;
                    if (live && d + e < a.D) store_f32(out + d + e, v);
                }
            }
            if (tiles > 0) {                          // O has been read: the next piece may use it
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.oempty[g]);
            }
            if (cut && live && half == 0) plan.ml[slot] = make_float2(ms, ls);
            if (!cut && live && half == 0 && a.lse != nullptr)
                a.lse[at * a.Hq + h] = ls > 0.0f ? (ms + __log2f(ls)) * ATT_LN2 : -INFINITY;
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

// Adds the shares of the cut pieces: weights 2^(m_s - max m), 32 shares at a time, then a warp's lanes hold DP / 32
// elements each. Every warp reads the records and takes one row in `step` of those that they name (a block per
// piece and some rows spent 20 us on 11520 blocks with nothing to do, where 192 pieces had not been cut).
constexpr int AF_JOIN_WARPS = 16;
template <typename T, int DP>
DN8_DEV void join_row(const dn8_attention_args& a, const TilePlan& plan, int block, int cuts, int64_t row, int r) {
    const int lane = threadIdx.x & 31, h = block % a.Hq;
    // (share s of the same piece and head: block + s Hq)
    auto slot = [&](int s) { return (static_cast<int64_t>(block) + static_cast<int64_t>(s) * a.Hq) * (2 * AT_TILE) + r; };
    float mm = -INFINITY, lv = 0.0f, ov[DP / 32] = {};
    for (int s = lane; s < cuts; s += 32) mm = fmaxf(mm, plan.ml[slot(s)].x);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, k));
    const float ref = mm == -INFINITY ? 0.0f : mm;
    for (int s0 = 0; s0 < cuts; s0 += 32) {
        float w = 0.0f;
        if (s0 + lane < cuts) {
            const float2 ml = plan.ml[slot(s0 + lane)];
            w = ex2(ml.x - ref);
            lv = fmaf(w, ml.y, lv);
        }
        const int ns = min(32, cuts - s0);
#pragma unroll 8
        for (int s = 0; s < ns; ++s) {
            float v[DP / 32];
            load_f32(plan.o + slot(s0 + s) * DP + lane * (DP / 32), v);
            const float ws = __shfl_sync(0xffffffffu, w, s);
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) ov[e] = fmaf(ws, v[e], ov[e]);
        }
    }
    lv = warp_sum(lv);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) ov[e] = lv > 0.0f ? ov[e] / lv : 0.0f;
    if (lane * (DP / 32) < a.D)
        store_f32(static_cast<T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h + lane * (DP / 32), ov);
    if (lane == 0 && a.lse != nullptr) a.lse[row * a.Hq + h] = lv > 0.0f ? (mm + log2f(lv)) * ATT_LN2 : -INFINITY;
}
template <typename T, int DP>
__global__ void __launch_bounds__(AF_JOIN_WARPS * 32) attn_tile_join_kernel(const dn8_attention_args a, const TilePlan plan) {
    constexpr int BATCH = 4;                          // 32 records each, loaded together
    const int lane = threadIdx.x & 31, blocks = plan.units * a.Hq, step = gridDim.x * AF_JOIN_WARPS;
    int next = blockIdx.x * AF_JOIN_WARPS + (threadIdx.x >> 5), run = 0;
    griddep_wait();
    for (int base = 0; base < blocks; base += 32 * BATCH) {
        int4 rec[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int block = base + 32 * x + lane;
            rec[x] = block < blocks ? plan.rec[block] : make_int4(0, 0, 0, 0);
            // (offsets that go back and forth may ask for more shares than there is room for, and a kernel that gave
            // up leaves records behind that say nothing: rows and shares are kept inside the tensors)
            rec[x].z = min(rec[x].z, (blocks - 1 - block) / a.Hq + 1);
            if (rec[x].x < 0 || rec[x].y < 0 || rec[x].y > 2 * AT_TILE || static_cast<int64_t>(rec[x].x) + rec[x].y > a.Tq)
                rec[x].y = 0;
        }
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            int incl = rec[x].y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const int total = __shfl_sync(0xffffffffu, incl, 31);
            for (; next < run + total; next += step) {
                const int src = __ffs(__ballot_sync(0xffffffffu, next < run + incl)) - 1;
                const int r = next - run - __shfl_sync(0xffffffffu, incl - rec[x].y, src);
                const int64_t row = static_cast<int64_t>(__shfl_sync(0xffffffffu, rec[x].x, src)) + r;
                join_row<T, DP>(a, plan, base + 32 * x + src, __shfl_sync(0xffffffffu, rec[x].z, src), row, r);
            }
            run += total;
        }
    }
}

// (a bound on the pieces: every sequence may leave one unfilled)
static int64_t tile_pieces(const dn8_attention_args& a) { return a.Tq / (2 * AT_TILE) + (a.B < a.Tq ? a.B : a.Tq); }
static TilePlan tile_plan(const dn8_attention_args& a, int sms) {
    TilePlan p = {};
    const int64_t pieces = tile_pieces(a);
    if (a.Tq * a.Hq < sms * AT_TILE && pieces * a.Hq < 2ll * sms && a.Tk >= 2 * AF_SHARE * AT_TILE) {
        p.sms = sms;
        // sum of max(1, tiles / part) <= pieces + sms / Hq (and one for the rounding of the sums)
        p.units = static_cast<int>(pieces) + sms / a.Hq + 1;
    }
    return p;
}
size_t attention_tile_work(const dn8_attention_args& a, int sms) {
    return static_cast<size_t>(tile_plan(a, sms).units) * a.Hq * 2 * AT_TILE * ((a.D <= 64 ? 64 : 128) + 2) * sizeof(float) +
           static_cast<size_t>(tile_plan(a, sms).units) * a.Hq * sizeof(int4);
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

template <typename T, int DP> static cudaError_t tile_go(const dn8_attention_args& a, int sms, cudaStream_t st) {
    CUtensorMap mq = {}, mk = {}, mv = {};
    cudaError_t e = make_head_map(&mq, a.q, a.type, a.Tq, a.Hq, a.D, a.q_stride_t, a.q_stride_h);
    if (e == cudaSuccess && a.Tk > 0) e = make_head_map(&mk, a.k, a.type, a.Tk, a.Hk, a.D, a.k_stride_t, a.k_stride_h);
    if (e == cudaSuccess && a.Tk > 0) e = make_head_map(&mv, a.v, a.type, a.Tk, a.Hk, a.D, a.v_stride_t, a.v_stride_h);
    if (e != cudaSuccess) return e;
    TilePlan plan = tile_plan(a, sms);
    const auto kernel = plan.sms > 0 ? attn_tile_kernel<T, DP, true> : attn_tile_kernel<T, DP, false>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    const int64_t blocks = (plan.sms > 0 ? plan.units : tile_pieces(a)) * a.Hq;
    if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    plan.o = static_cast<float*>(a.work);
    plan.ml = reinterpret_cast<float2*>(plan.o + blocks * 2 * AT_TILE * DP);
    plan.rec = reinterpret_cast<int4*>(plan.ml + blocks * 2 * AT_TILE);
    e = launch_pdl(false, kernel, dim3(static_cast<unsigned>(blocks)), dim3(AF_THREADS), TileCfg<DP>::SMEM,
                   st, mq, mk, mv, a, plan);
    if (e != cudaSuccess || plan.sms == 0) return e;
    return launch_pdl(true, attn_tile_join_kernel<T, DP>, dim3(2 * sms), dim3(AF_JOIN_WARPS * 32), 0, st, a, plan);
}

cudaError_t launch_attention_tile(const dn8_attention_args& a, int sms, cudaStream_t st) {
    if (a.type == DN8_F16) return a.D <= 64 ? tile_go<__half, 64>(a, sms, st) : tile_go<__half, 128>(a, sms, st);
    return a.D <= 64 ? tile_go<__nv_bfloat16, 64>(a, sms, st) : tile_go<__nv_bfloat16, 128>(a, sms, st);
}

}  // namespace dn8
