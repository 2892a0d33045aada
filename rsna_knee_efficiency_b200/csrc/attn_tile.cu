// attn_tile.cu -- attention of many query rows on the tensor cores.
//
// One CTA = up to 256 query rows of one head of one sequence, as two tiles of 128 rows, over the key tiles
// that some row of them sees. Per key tile and query tile:
//   S = Q K^T        tcgen05 128 x 128 x D into TMEM,
//   P = 2^(S c - m)  one thread per row reads S from TMEM; P goes back to TMEM in 16 bits, over S,
//   O += P V         tcgen05 128 x D x 128, P from TMEM, V as it lies in memory.
// Two query tiles alternate: while the threads of one take the exponentials of their S, the tensor cores
// work on the other. The reference m of a row is its running maximum at the time of the last
// rescaling: O and the sum are rescaled only when the maximum has grown by more than 2^8 (then P <=
// 256, far inside fp16 and fp32), so the accumulator rarely leaves TMEM.
//
// Warps 0-3 and 4-7: softmax of tile 0 and 1, then the output. Warp 8: tcgen05 issue. Warp 9: TMA. Warp 10:
// rows of V that nobody may see (behind the sequence, keep = 0) are zeroed in shared memory before the
// product, since 0 * NaN is not 0 (their scores are replaced, so K may hold anything).
#include "attn_umma.cuh"

namespace dn8 {

constexpr int AF_THREADS = 384;
// The launch gives every thread 168 registers (12 warps); a softmax thread holds a row of 128 scores and
// more, the other four warps little: 8 x 32 x 208 + 4 x 32 x 88 = 12 x 32 x 168.
constexpr int AF_REGS_SOFTMAX = 208, AF_REGS_OTHER = 88;

template <int DP> struct TileCfg {
    static constexpr int KST = DP == 64 ? 3 : 2, VST = DP == 64 ? 3 : 2;      // stages of K and V
    static constexpr uint32_t TILE = AT_TILE * DP * 2;
    static constexpr uint32_t SMEM = 1024 + TILE * (2 + KST + VST) + 1024;
    // TMEM columns: S (and P) of the two tiles, O of the two tiles
    static constexpr uint32_t S0 = 0, O0 = 256;
};

struct TileShared {
    uint64_t qfull, fin;
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], vok[3];
    uint64_t sfull[2], pfull[2];
    uint32_t words[3][4];
    uint32_t tmem;
    int abort;
    Sequence seq;
};

template <typename T, int DP>
__global__ void __launch_bounds__(AF_THREADS, 1)
attn_tile_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const dn8_attention_args a) {
    using C = TileCfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = smem;
    uint8_t* sk = sq + 2 * C::TILE;
    uint8_t* sv = sk + C::KST * C::TILE;
    TileShared& sh = *reinterpret_cast<TileShared*>(sv + C::VST * C::TILE);
    volatile int* abort_flag = &sh.abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.Hq, kvh = h / (a.Hq / a.Hk);
    if (warp == 8) {
        const Sequence f = find_block<false>(a, blockIdx.x / a.Hq, 1, 2 * AT_TILE);
        if (lane == 0) {
            sh.seq = f;
            mbar_init(&sh.qfull, 1);
            mbar_init(&sh.fin, 1);
            for (int s = 0; s < 3; ++s) {
                mbar_init(&sh.kfull[s], 1);
                mbar_init(&sh.kempty[s], 1);
                mbar_init(&sh.vfull[s], 1);
                mbar_init(&sh.vempty[s], 2);        // the product and warp 10
                mbar_init(&sh.vok[s], 1);
            }
            for (int g = 0; g < 2; ++g) {
                mbar_init(&sh.sfull[g], 1);
                mbar_init(&sh.pfull[g], 4);
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
    // last blocks first: with an open left side they are the longest
    const int i0 = seq.b < 0 ? 0 : ((seq.nq - 1) / (2 * AT_TILE) - seq.blk) * 2 * AT_TILE;
    KeyTiles all, own[2];
    all.count = own[0].count = own[1].count = 0;
    if (seq.b >= 0) {
        all = key_tiles(i0 + off, min(i0 + 2 * AT_TILE, seq.nq) - 1 + off, seq.nk, left, right, a.sinks, AT_TILE);
#pragma unroll
        for (int g = 0; g < 2; ++g)
            if (i0 + g * AT_TILE < seq.nq)
                own[g] = key_tiles(i0 + g * AT_TILE + off, min(i0 + (g + 1) * AT_TILE, seq.nq) - 1 + off, seq.nk, left,
                                   right, a.sinks, AT_TILE);
    }
    // tile `t` is one of query tile g's own
    auto uses = [&](int g, int t) -> bool {
        return own[g].count > 0 && (t < own[g].first || (t >= own[g].start && t < own[g].start + own[g].count - own[g].first));
    };
    // V of tile t has rows to zero
    auto fixed = [&](int t) -> bool { return a.keep != nullptr || (t + 1) * AT_TILE > seq.nk; };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AF_REGS_OTHER));
        if (all.count == 0) {
            // nothing to do
        } else if (warp == 9) {
            // ---------------- TMA ----------------
            if (lane == 0) {
                const int nt = i0 + AT_TILE < seq.nq ? 2 : 1;
                mbar_expect_tx(&sh.qfull, nt * C::TILE);
                for (int g = 0; g < nt; ++g)
                    load_tile<DP>(sq + g * C::TILE, &mq, &sh.qfull, h, seq.q0 + i0 + g * AT_TILE);
                for (int u = 0; u < all.count; ++u) {
                    const int row = seq.k0 + all.tile(u) * AT_TILE, ks = u % C::KST, vs = u % C::VST;
                    if (!mbar_wait(&sh.kempty[ks], ((u / C::KST) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (64 << 4))) break;
                    mbar_expect_tx(&sh.kfull[ks], C::TILE);
                    load_tile<DP>(sk + ks * C::TILE, &mk, &sh.kfull[ks], kvh, row);
                    if (!mbar_wait(&sh.vempty[vs], ((u / C::VST) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (65 << 4))) break;
                    mbar_expect_tx(&sh.vfull[vs], C::TILE);
                    load_tile<DP>(sv + vs * C::TILE, &mv, &sh.vfull[vs], kvh, row);
                }
            }
            __syncwarp();
        } else if (warp == 10) {
            // ---------------- masked rows of V ----------------
            for (int u = 0; u < all.count; ++u) {
                const int t = all.tile(u), vs = u % C::VST;
                const bool fix = fixed(t);
                uint32_t word[4];
                if (fix)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int j = t * AT_TILE + w * 32 + lane;
                        word[w] = __ballot_sync(0xffffffffu, j < seq.nk && (a.keep == nullptr || a.keep[seq.k0 + j] != 0));
                    }
                // (every tile is waited for, and its stage released here too, so that this warp keeps step)
                if (!mbar_wait_w(&sh.vfull[vs], (u / C::VST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (66 << 4))) break;
                if (fix) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if (lane == w) sh.words[vs][w] = word[w];
                        if (!((word[w] >> lane) & 1u))
#pragma unroll
                            for (int b = 0; b < DP / 64; ++b) {
                                uint4* row = reinterpret_cast<uint4*>(sv + vs * C::TILE + b * AT_BLOCK + (w * 32 + lane) * 128);
#pragma unroll
                                for (int c = 0; c < 8; ++c) row[c] = make_uint4(0u, 0u, 0u, 0u);
                            }
                    }
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0) {
                    if (fix) mbar_arrive(&sh.vok[vs]);
                    mbar_arrive(&sh.vempty[vs]);
                }
            }
        } else if (warp == 8) {
            // ---------------- tcgen05 issue ----------------
            const uint32_t q0 = smem_u32(sq), k0 = smem_u32(sk), v0 = smem_u32(sv);
            int np[2] = {0, 0};                       // products O += P V issued per query tile
            bool ok = mbar_wait_w(&sh.qfull, 0, a.err, abort_flag, ERR_WAIT_FULL | (67 << 4));
            for (int u = 0; ok && u <= all.count; ++u) {
                const int ks = u % C::KST, vp = (u - 1) % C::VST;
                if (u < all.count) {
                    ok = mbar_wait_w(&sh.kfull[ks], (u / C::KST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (68 << 4));
                    if (!ok) break;
                }
                if (u > 0) {
                    const int w = (u - 1) / C::VST;
                    ok = mbar_wait_w(&sh.vfull[vp], w & 1, a.err, abort_flag, ERR_WAIT_FULL | (69 << 4));
                    // (without a mask only the last tile is fixed: its barrier's first phase)
                    if (ok && fixed(all.tile(u - 1)))
                        ok = mbar_wait_w(&sh.vok[vp], a.keep != nullptr ? w & 1 : 0, a.err, abort_flag,
                                         ERR_WAIT_FULL | (70 << 4));
                    if (!ok) break;
                }
                tc_fence_after();
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    if (u > 0 && uses(g, all.tile(u - 1))) {
                        ok = mbar_wait_w(&sh.pfull[g], np[g] & 1, a.err, abort_flag, ERR_WAIT_ACC | (71 << 4));
                        if (!ok) break;
                        tc_fence_after();
                        mma_values<T, DP>(tmem + C::O0 + g * DP, tmem + C::S0 + g * 128, v0 + vp * C::TILE, np[g] > 0);
                        ++np[g];
                    }
                    if (u < all.count && uses(g, all.tile(u))) {
                        // (S lies over P: the product that reads P was issued before)
                        mma_scores<T, DP>(tmem + C::S0 + g * 128, q0 + g * C::TILE, k0 + ks * C::TILE);
                        umma_commit_w(&sh.sfull[g]);
                    }
                }
                if (u < all.count) umma_commit_w(&sh.kempty[ks]);
                if (u > 0) umma_commit_w(&sh.vempty[vp]);
            }
            if (ok) umma_commit_w(&sh.fin);
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AF_REGS_SOFTMAX));
        if (seq.b >= 0) {
        // ---------------- softmax: one row per thread ----------------
        const int g = warp >> 2, row = (warp & 3) * 32 + lane;
        const int i = i0 + g * AT_TILE + row, p = i + off;
        const uint32_t quad = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + C::S0 + g * 128 + quad, to = tmem + C::O0 + g * DP + quad;
        const float sc = a.scale * ATT_LOG2E;
        // positions of the tile's first and last row, for tiles that need no mask
        const int pa = i0 + g * AT_TILE + off, pb = min(i0 + (g + 1) * AT_TILE, seq.nq) - 1 + off;
        float m = -INFINITY, l = 0.0f;               // reference (times sc) and sum
        int n = 0;
        bool ok = true;
        for (int u = 0; u < all.count; ++u) {
            const int t = all.tile(u), j0 = t * AT_TILE;
            if (!uses(g, t)) continue;
            uint32_t word[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
            const int last = j0 + AT_TILE - 1;
            const bool masked = a.keep != nullptr || last > min(seq.nk - 1, pa + right) || (j0 < pb - left && last >= a.sinks);
            if (masked) {
                if (a.keep != nullptr) {
                    ok = mbar_wait_w(&sh.vok[u % C::VST], (u / C::VST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (72 << 4));
                    if (!ok) break;
                }
                const int hi = min(seq.nk - 1, p + right) - j0, lo = p - left - j0;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    word[w] = bits_upto(hi, w) & (bits_from(lo, w) | bits_upto(a.sinks - 1 - j0, w)) &
                              (a.keep != nullptr ? sh.words[u % C::VST][w] : 0xFFFFFFFFu);
            }
            ok = mbar_wait_w(&sh.sfull[g], n & 1, a.err, abort_flag, ERR_WAIT_ACC | (73 << 4));
            if (!ok) break;
            tc_fence_after();
            uint32_t r[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, r[c]);
            tmem_wait_ld(r[0]);
            reg_bind(r[1]);
            reg_bind(r[2]);
            reg_bind(r[3]);
            if (masked)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[c][e] = (word[c] >> e) & 1u ? r[c][e] : 0xFF800000u;   // -inf
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(r[c][e]));
            mx *= sc;
            if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                const float mn = fmaxf(m, mx);
                const float f = ex2(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= f;
                if (n > 0) {
                    // S complete: so is the product before it, and the next one waits for P
#pragma unroll
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(to + 32 * c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(to + 32 * c, o);
                        tmem_wait_st(o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            const float2 sc2 = f2_pack(sc, sc), mr2 = f2_pack(-ref, -ref);
            float2 s2 = f2_pack(0.0f, 0.0f);
            uint32_t pk[4][16];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 x = f2_fma(f2_pack(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), sc2, mr2);
                    x.x = ex2(x.x);
                    x.y = ex2(x.y);
                    s2 = __fadd2_rn(s2, x);
                    // the weights are rounded to the values' type, the type of the matrix instruction
                    pk[c][e] = pack2(T(), x.x, x.y);
                }
                tmem_st16(ts + 16 * c, pk[c]);
            }
            l += s2.x + s2.y;
            tmem_wait_st(pk[0]);
            tmem_wait_st(pk[1]);
            tmem_wait_st(pk[2]);
            tmem_wait_st(pk[3]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pfull[g]);
            ++n;
        }
        if (ok && n > 0) {
            ok = mbar_wait_w(&sh.fin, 0, a.err, abort_flag, ERR_WAIT_ACC | (74 << 4));
            tc_fence_after();
        }
        const int64_t at = seq.q0 + i;
        const bool live = ok && i < seq.nq;
        T* out = static_cast<T*>(a.out) + at * a.o_stride_t + static_cast<int64_t>(h) * a.o_stride_h;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            if (n > 0 && ok) {
                tmem_ld32(to + 32 * c, o);
                tmem_wait_ld(o);
            }
            if (live)
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    if (32 * c + e < a.D) {
                        float v[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) v[x] = l > 0.0f ? __uint_as_float(o[e + x]) * inv : 0.0f;
                        store_f32(out + 32 * c + e, v);
                    }
        }
        if (live && a.lse != nullptr) a.lse[at * a.Hq + h] = l > 0.0f ? (m + __log2f(l)) * ATT_LN2 : -INFINITY;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t make_head_map(CUtensorMap* map, const void* base, int type, int64_t rows, int heads, int D, int64_t stride_t,
                          int64_t stride_h) {
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
    cuuint32_t box[3] = {64, 1, AT_TILE};
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
