// attn.cu -- attention over packed sequences with a sliding window, first tokens that stay visible and
// a key mask; grouped heads.
#include "attn_umma.cuh"

namespace dn8 {

// ---- few rows over a long key axis -----------------------------------------------------------
// The query rows of one key head's group (row r = query r / G, head r % G of the group) in blocks of
// 16, one CTA per (row block, key head, share of the key tiles). Bound by reading keys and values once:
// every warp streams its own tiles (16 KB / D keys: 4 KB of keys, 4 KB of values) through its own ring of
// TMA stages (no barrier between warps), multiplies with 16-row matrix instructions (a tcgen05 tile has
// 128 rows, of which a single token with 4 heads per group would fill 4) and keeps its own running
// maximum, sum and output; the warps are joined in shared memory, the shares of the key axis by
// attn_join_kernel. Loads by cp.async with an address and a mask test per 16 bytes took 767 instructions
// per tile and left the memory half idle; a TMA tile takes one, and tests are made per tile.
// One token of each of 8 streams over caches of 1 to 32768 (551 MB of keys and values), 32 heads on 8, D = 128: 105 us,
// 5.2 TB/s, 0.81 of the copy rate; 4 queries over 16 x 12288 tokens, 8 heads, D = 64 (403 MB): 78 us, 5.1 TB/s.
// Rows of values that no query of the sequence may see (behind its end, keep = 0, or before every window) are zeroed
// in shared memory, since 0 * NaN is not 0; their scores are replaced, so keys may hold anything.
constexpr int AR_WARPS = 4, AR_ROWS = 16, AR_STAGES = 3;
constexpr uint32_t AR_TILE_BYTES = 4096, AR_STAGE = 2 * AR_TILE_BYTES;

DN8_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DN8_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> DN8_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> DN8_DEV void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> DN8_DEV void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Shares of a row block's key axis. Lengths are known to the GPU alone, so each CTA adds them up: every row block
// is cut into as many whole parts of 1 / slots of all keys as it holds, and the CTAs are numbered block by
// block, share by share, so that they run side by side and end together, however ragged the caches are.
// (Several waves of short shares cost a start and an end each: 16 x 12288 keys, 8 heads, 74 us in one wave, 79 in
// two, 90 in five.)
struct RowsPlan {
    int units;               // CTAs per key head, a bound: row blocks and shares
    int slots;               // CTAs per key head that the GPU holds at a time, or 0: nothing is cut
    float* ml;               // [key head][unit][16] (maximum in units of log2, sum)
    float* o;                // [key head][unit][16][DP], relative to the maximum
};
struct RowsShares {
    const dn8_attention_args& a;
    float part;              // keys
    DN8_DEV int operator()(int nq, int nk) const {
        return part > 0.0f ? max(1, static_cast<int>(seen_keys(a, nq, nk) / part)) : 1;
    }
};
template <int KEYS> DN8_DEV RowsShares rows_shares(const dn8_attention_args& a, const RowsPlan& plan) {
    RowsShares s = {a, 0.0f};                            // (one whole warp)
    if (plan.slots == 0) return s;
    const int G = a.Hq / a.Hk;
    float total = 0.0f;
    for (int b = threadIdx.x & 31; b < a.B; b += 32) {
        const Sequence q = sequence_of(a, b);
        total += static_cast<float>((static_cast<int64_t>(q.nq) * G + AR_ROWS - 1) / AR_ROWS) *
                 static_cast<float>(seen_keys(a, q.nq, q.nk));
    }
    s.part = fmaxf(warp_sum(total) / static_cast<float>(plan.slots), 4.0f * AR_WARPS * KEYS);
    return s;
}

template <typename T, int DP>
__global__ void __launch_bounds__(AR_WARPS * 32, 2)
attn_rows_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                 const dn8_attention_args a, const RowsPlan plan) {
    constexpr int KEYS = AR_TILE_BYTES / (DP * 2);       // keys of a tile
    constexpr uint32_t BLOCK = KEYS * 128;               // bytes of its 64 first elements
    extern __shared__ uint8_t sm_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Sequence s_seq;
    __shared__ uint64_t s_full[AR_WARPS][AR_STAGES];
    __shared__ int s_abort, s_shares;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk, kvh = blockIdx.y;
    griddep_launch_dependents();
    if (warp == 0) {
        const RowsShares cuts = rows_shares<KEYS>(a, plan);
        const Sequence f = find_block<false>(a, blockIdx.x, G, AR_ROWS, cuts);
        if (lane == 0) {
            s_seq = f;
            s_shares = f.b < 0 ? 1 : cuts(f.nq, f.nk);
        }
    } else if (threadIdx.x == 32) {
        for (int w = 0; w < AR_WARPS; ++w)
            for (int k = 0; k < AR_STAGES; ++k) mbar_init(&s_full[w][k], 1);
        s_abort = 0;
        mbar_fence_init();
    }
    __syncthreads();
    const Sequence sq = s_seq;
    if (sq.b < 0) return;
    const int shares = s_shares, share = sq.blk % shares;
    volatile int* abort_flag = &s_abort;
    const int r0 = sq.blk / shares * AR_ROWS, nrows = min(AR_ROWS, sq.nq * G - r0);
    const int off = sq.nk - sq.nq;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const int p0 = r0 / G + off, p1 = (r0 + nrows - 1) / G + off;      // first and last row's position
    const KeyTiles kt = key_tiles(p0, p1, sq.nk, left, right, a.sinks, KEYS);
    const int workers = shares * AR_WARPS, me = share * AR_WARPS + warp;
    uint8_t* ring = sm + warp * AR_STAGES * AR_STAGE;

    auto issue = [&](int t, int stage) {                 // (lane 0)
        if (t >= kt.count) return;
        const int row = sq.k0 + kt.tile(t) * KEYS;
        uint8_t* dst = ring + stage * AR_STAGE;
        mbar_expect_tx(&s_full[warp][stage], AR_STAGE);
#pragma unroll
        for (int b = 0; b < DP / 64; ++b) {
            tma_load_3d(dst + b * BLOCK, &mk, &s_full[warp][stage], b * 64, kvh, row);
            tma_load_3d(dst + AR_TILE_BYTES + b * BLOCK, &mv, &s_full[warp][stage], b * 64, kvh, row);
        }
    };
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < AR_STAGES; ++k) issue(me + k * workers, k);

    // the queries as matrix-instruction fragments
    uint32_t qf[DP / 16][4];
    int pos[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = r0 + lane / 4 + 8 * half;
        const bool live = lane / 4 + 8 * half < nrows;
        pos[half] = r / G + off;
        const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(sq.q0 + r / G) * a.q_stride_t +
                     static_cast<int64_t>(kvh * G + r % G) * a.q_stride_h;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int d = kk * 16 + c * 8 + (lane & 3) * 2;
                qf[kk][half + 2 * c] = live && d < a.D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
            }
    }
    const uint32_t hidden = hidden_keys(a, sq.nq, sq.nk);
    auto kept = [&](int t) -> bool {                     // this lane's key of tile index t may be seen
        if (t >= kt.count || lane >= KEYS) return true;
        const int j = kt.tile(t) * KEYS + lane;
        return j < sq.nk && behind_hidden(a, j, hidden) && (a.keep == nullptr || a.keep[sq.k0 + j] != 0);
    };
    bool next_kept = kept(me);

    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};          // references (times sc) and sums
    const float sc = a.scale * ATT_LOG2E;
    const int mat = lane >> 3, mr = lane & 7;
    int stage = 0, phase = 0;
    for (int t = me; t < kt.count; t += workers) {
        const uint32_t word = __ballot_sync(0xffffffffu, next_kept);
        next_kept = kept(t + workers);
        if (!mbar_wait_w(&s_full[warp][stage], phase, a.err, abort_flag, ERR_WAIT_FULL | (57 << 4))) break;
        uint8_t* tile = ring + stage * AR_STAGE;
        const uint32_t kb = smem_u32(tile), vb = kb + AR_TILE_BYTES;
        const int j0 = kt.tile(t) * KEYS;
        if (word != 0xFFFFFFFFu) {
            if (!((word >> lane) & 1u))
#pragma unroll
                for (int b = 0; b < DP / 64; ++b)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        reinterpret_cast<uint4*>(tile + AR_TILE_BYTES + b * BLOCK + lane * 128)[c] = make_uint4(0u, 0u, 0u, 0u);
            fence_async_smem();                          // (before the stage's next load)
            __syncwarp();
        }
        float s[KEYS / 8][4];
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int np = 0; np < KEYS / 16; ++np) {
                uint32_t b[4];
                const int key = np * 16 + (mat >> 1) * 8 + mr, ch = (kk & 3) * 2 + (mat & 1);
                ldsm4(b, kb + (kk >> 2) * BLOCK + key * 128 + ((ch ^ (key & 7)) << 4));
                mma16<T>(s[2 * np], qf[kk], b[0], b[1]);
                mma16<T>(s[2 * np + 1], qf[kk], b[2], b[3]);
            }
        // does every row see every key of the tile?
        if (word != 0xFFFFFFFFu || j0 + KEYS - 1 > p0 + right || (j0 < p1 - left && j0 + KEYS > a.sinks))
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int jl = n * 8 + (lane & 3) * 2 + (e & 1), j = j0 + jl, p = pos[e >> 1];
                    const bool see = ((word >> jl) & 1u) && j <= p + right && (j >= p - left || j < a.sinks);
                    s[n][e] = see ? s[n][e] : -INFINITY;
                }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)) * sc;
        }
        // (rescaled only when a maximum has grown by more than 2^8: the weights stay below 256)
        if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.0f || mx[1] > m[1] + 8.0f))
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float mn = fmaxf(m[h], mx[h]);
                const float f = ex2(m[h] - (mn == -INFINITY ? 0.0f : mn));
                m[h] = mn;
                l[h] *= f;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][2 * h] *= f;
                    o[n][2 * h + 1] *= f;
                }
            }
        const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = ex2(fmaf(s[n][e], sc, -ref[e >> 1]));
                l[e >> 1] += s[n][e];
            }
#pragma unroll
        for (int kp = 0; kp < KEYS / 16; ++kp) {
            // weights rounded to the values' type, the type of the matrix instruction
            const uint32_t p[4] = {pack2(T(), s[2 * kp][0], s[2 * kp][1]), pack2(T(), s[2 * kp][2], s[2 * kp][3]),
                                   pack2(T(), s[2 * kp + 1][0], s[2 * kp + 1][1]),
                                   pack2(T(), s[2 * kp + 1][2], s[2 * kp + 1][3])};
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                const int key = kp * 16 + (mat & 1) * 8 + mr, ch = (n & 3) * 2 + (mat >> 1);
                ldsm4t(b, vb + (n >> 2) * BLOCK + key * 128 + ((ch ^ (key & 7)) << 4));
                mma16<T>(o[2 * n], p, b[0], b[1]);
                mma16<T>(o[2 * n + 1], p, b[2], b[3]);
            }
        }
        __syncwarp();                                    // every lane has read the stage
        if (lane == 0) issue(t + AR_STAGES * workers, stage);
        if (++stage == AR_STAGES) {
            stage = 0;
            phase ^= 1;
        }
    }
    __syncthreads();                                     // the rings are free: join the warps there
    if (*abort_flag) return;
    float* so = reinterpret_cast<float*>(sm);            // [warp][16][DP]
    float* sml = so + AR_WARPS * AR_ROWS * DP;           // [warp][16][2]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = lane / 4 + 8 * h;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2*>(so + (warp * AR_ROWS + r) * DP + n * 8 + (lane & 3) * 2) =
                make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if ((lane & 3) == 0) {
            sml[(warp * AR_ROWS + r) * 2] = m[h];
            sml[(warp * AR_ROWS + r) * 2 + 1] = l[h];
        }
    }
    __syncthreads();
    const size_t slot = static_cast<size_t>(kvh) * plan.units + blockIdx.x;
    for (int k = threadIdx.x; k < nrows * DP; k += AR_WARPS * 32) {
        const int r = k / DP, d = k % DP;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < AR_WARPS; ++w) mm = fmaxf(mm, sml[(w * AR_ROWS + r) * 2]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ov = 0.0f, lv = 0.0f;
#pragma unroll
        for (int w = 0; w < AR_WARPS; ++w) {
            const float f = ex2(sml[(w * AR_ROWS + r) * 2] - ref);
            ov = fmaf(f, so[(w * AR_ROWS + r) * DP + d], ov);
            lv = fmaf(f, sml[(w * AR_ROWS + r) * 2 + 1], lv);
        }
        if (shares > 1) {
            plan.o[(slot * AR_ROWS + r) * DP + d] = ov;
            if (d == 0) {
                plan.ml[(slot * AR_ROWS + r) * 2] = mm;
                plan.ml[(slot * AR_ROWS + r) * 2 + 1] = lv;
            }
            continue;
        }
        const int64_t row = sq.q0 + (r0 + r) / G;
        const int h = kvh * G + (r0 + r) % G;
        if (d < a.D)
            (static_cast<T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h)[d] = from_f32<T>(lv > 0.0f ? ov / lv : 0.0f);
        if (d == 0 && a.lse != nullptr) a.lse[row * a.Hq + h] = lv > 0.0f ? (mm + log2f(lv)) * ATT_LN2 : -INFINITY;
    }
}

// Adds the shares of a row block, one warp per row: weights 2^(m_s - max m), a share per lane (32 at a
// time), then the lanes hold DP / 32 elements each and read the shares' rows.
template <typename T, int DP>
__global__ void __launch_bounds__(AR_ROWS * 32) attn_join_kernel(const dn8_attention_args a, const RowsPlan plan) {
    __shared__ Sequence s_seq;
    __shared__ int s_shares;
    const int G = a.Hq / a.Hk, kvh = blockIdx.y, r = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (r == 0) {
        const auto cuts = rows_shares<AR_TILE_BYTES / (DP * 2)>(a, plan);
        const Sequence f = find_block<false>(a, blockIdx.x, G, AR_ROWS, cuts);
        if (lane == 0) {
            s_seq = f;
            s_shares = f.b < 0 ? 1 : cuts(f.nq, f.nk);
        }
    }
    __syncthreads();
    const Sequence sq = s_seq;
    const bool idle = sq.b < 0 || s_shares <= 1 || sq.blk % s_shares != 0;      // (one share: the output is written)
    // A block with nothing to add leaves without waiting, and its room goes to one that has (where all wait, a token
    // over each of 8 caches takes 109 us, not 105). But the first one always waits: were all to leave (nothing is cut),
    // this grid would be over, and what comes after it let go, while the row kernel still writes.
    if (!idle || (blockIdx.x == 0 && blockIdx.y == 0)) griddep_wait();
    if (idle) return;
    const int rr = sq.blk / s_shares * AR_ROWS + r;
    if (rr >= sq.nq * G) return;
    // (offsets that go back and forth may ask for more shares than there is room for)
    const int shares = min(s_shares, plan.units - static_cast<int>(blockIdx.x));
    const size_t slot = static_cast<size_t>(kvh) * plan.units + blockIdx.x;
    float mm = -INFINITY;
    for (int s = lane; s < shares; s += 32) mm = fmaxf(mm, plan.ml[((slot + s) * AR_ROWS + r) * 2]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, k));
    const float ref = mm == -INFINITY ? 0.0f : mm;
    float lv = 0.0f, ov[DP / 32] = {};
    for (int s0 = 0; s0 < shares; s0 += 32) {
        float w = 0.0f;
        if (s0 + lane < shares) {
            const float2 ml = *reinterpret_cast<const float2*>(plan.ml + ((slot + s0 + lane) * AR_ROWS + r) * 2);
            w = ex2(ml.x - ref);
            lv = fmaf(w, ml.y, lv);
        }
        const int ns = min(32, shares - s0);
#pragma unroll 8
        for (int s = 0; s < ns; ++s) {
            float v[DP / 32];
            load_f32(plan.o + ((slot + s0 + s) * AR_ROWS + r) * DP + lane * (DP / 32), v);
            const float ws = __shfl_sync(0xffffffffu, w, s);
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) ov[e] = fmaf(ws, v[e], ov[e]);
        }
    }
    lv = warp_sum(lv);
    const int64_t row = sq.q0 + rr / G;
    const int h = kvh * G + rr % G;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) ov[e] = lv > 0.0f ? ov[e] / lv : 0.0f;
    if (lane * (DP / 32) < a.D) store_f32(static_cast<T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h + lane * (DP / 32), ov);
    if (lane == 0 && a.lse != nullptr) a.lse[row * a.Hq + h] = lv > 0.0f ? (mm + log2f(lv)) * ATT_LN2 : -INFINITY;
}

namespace {

int head_pad(int D) { return D <= 64 ? 64 : 128; }

// Row blocks (a bound: every sequence may leave one block unfilled), and shares: the sum of max(1, keys / part) is
// at most blocks + slots (and one for the rounding of the sums). Many row blocks fill the GPU uncut.
RowsPlan rows_plan(const dn8_attention_args& a, int sms) {
    RowsPlan p = {};
    const int64_t rows = a.Tq * (a.Hq / a.Hk);
    const int64_t blocks = rows / AR_ROWS + (a.B < rows ? a.B : rows);
    const int64_t slots = 2 * sms / a.Hk;                // (two CTAs per SM, by their shared memory)
    p.units = static_cast<int>(blocks);
    if (slots > 0 && blocks < 4 * slots && a.Tk * head_pad(a.D) * 2 / AR_TILE_BYTES >= 8 * AR_WARPS) {
        p.slots = static_cast<int>(slots);
        p.units = static_cast<int>(blocks + slots + 1);
    }
    return p;
}
size_t rows_work(const dn8_attention_args& a, const RowsPlan& p) {
    if (p.slots == 0) return 0;
    return static_cast<size_t>(p.units) * a.Hk * AR_ROWS * (head_pad(a.D) + 2) * sizeof(float);
}

template <typename T, int DP> cudaError_t rows_go(const dn8_attention_args& a, RowsPlan p, cudaStream_t st) {
    constexpr size_t ring = static_cast<size_t>(AR_WARPS) * AR_STAGES * AR_STAGE;
    constexpr size_t join = static_cast<size_t>(AR_WARPS) * AR_ROWS * (DP + 2) * 4;
    constexpr size_t smem = 1024 + (ring > join ? ring : join);
    cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    CUtensorMap mk = {}, mv = {};
    constexpr int keys = AR_TILE_BYTES / (DP * 2);
    if (a.Tk > 0) {
        e = make_head_map(&mk, a.k, a.type, a.Tk, a.Hk, a.D, a.k_stride_t, a.k_stride_h, keys);
        if (e == cudaSuccess) e = make_head_map(&mv, a.v, a.type, a.Tk, a.Hk, a.D, a.v_stride_t, a.v_stride_h, keys);
        if (e != cudaSuccess) return e;
    }
    if (p.slots > 0) {
        p.o = static_cast<float*>(a.work);
        p.ml = p.o + static_cast<size_t>(p.units) * a.Hk * AR_ROWS * DP;
    }
    e = launch_pdl(false, attn_rows_kernel<T, DP>, dim3(p.units, a.Hk), dim3(AR_WARPS * 32), smem, st, mk, mv, a, p);
    if (e != cudaSuccess || p.slots == 0) return e;
    return launch_pdl(true, attn_join_kernel<T, DP>, dim3(p.units, a.Hk), dim3(AR_ROWS * 32), 0, st, a, p);
}

}  // namespace

// Few rows per sequence and key head: the row kernel, which packs the heads of a group. Otherwise 128-row tiles on
// the tensor cores (attn_tile.cu). A tile costs about as much however few of its rows are used, a block of 16 rows
// reads all keys again (from L2) and pays a start and an end: up to 32 rows the row kernel, above that where
// the keys are many. 16 heads in groups of 4, D = 64, row kernel and tiles: 48 rows over 24 x 2000 keys 35 and 74
// us, over 64 x 500 52 and 62; 128 rows over 8 x 6000 51 and 77, over 24 x 2000 72 and 74, over 64 x 500 72 and 63;
// 256 rows over 8 x 6000 90 and 78. 8 heads, 48 rows over 200 x 200 keys: 168 and 74.
static bool few_rows(const dn8_attention_args& a) {
    const int64_t rows = a.Tq * (a.Hq / a.Hk);
    return rows <= 32ll * a.B || (rows <= 128ll * a.B && a.Tk >= 8 * rows);
}

size_t attention_work(const dn8_attention_args& a, int sms) {
    return few_rows(a) ? rows_work(a, rows_plan(a, sms)) : attention_tile_work(a, sms);
}

cudaError_t launch_attention(const dn8_attention_args& a, int sms, cudaStream_t st) {
    if (!few_rows(a)) return launch_attention_tile(a, sms, st);
    const RowsPlan p = rows_plan(a, sms);
    if (a.type == DN8_F16) return head_pad(a.D) == 64 ? rows_go<__half, 64>(a, p, st) : rows_go<__half, 128>(a, p, st);
    return head_pad(a.D) == 64 ? rows_go<__nv_bfloat16, 64>(a, p, st) : rows_go<__nv_bfloat16, 128>(a, p, st);
}

}  // namespace dn8
