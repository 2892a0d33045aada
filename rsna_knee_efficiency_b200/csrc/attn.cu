// attn.cu -- attention over packed sequences with a sliding window, first tokens that stay visible and
// a key mask; grouped heads.
#include "attn_umma.cuh"

namespace dn8 {

// ---- few rows over a long key axis -----------------------------------------------------------
// The query rows of one key head's group (row r = query r / G, head r % G of the group) in blocks of
// 16, one CTA per (row block, key head, share of the key tiles). Bound by reading keys and values once:
// every warp streams its own tiles of 32 keys through its own ring of cp.async stages (no barrier
// between warps), multiplies with 16-row matrix instructions (a tcgen05 tile has 128 rows, of which a
// single token with 4 heads per group would fill 4) and keeps its own running maximum, sum and output;
// the warps are joined in shared memory, the shares of the key axis by attn_join_kernel.
// Rows of keys and values that no query may see (behind the sequence's end, or keep = 0) are filled
// with zeros on the way in, so whatever they hold never meets an arithmetic instruction.
constexpr int AR_WARPS = 4, AR_ROWS = 16, AR_KEYS = 32, AR_STAGES = 3;

DN8_DEV void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
DN8_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> DN8_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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
// Where a share's partial results are kept: [row block][key head][share] of (16 rows x (maximum, sum)) and
// 16 x DP outputs, relative to the row's maximum (in units of log2).
struct RowsPlan {
    int blocks, splits;
    float* ml;
    float* o;
};

template <typename T, int DP>
__global__ void __launch_bounds__(AR_WARPS * 32) attn_rows_kernel(const dn8_attention_args a, const RowsPlan plan) {
    constexpr int CH = DP / 8;                           // 16-byte chunks of a row
    constexpr int STAGE = 2 * AR_KEYS * DP * 2;          // keys and values of a stage, bytes
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ Sequence s_seq;
    __shared__ uint32_t s_words[AR_WARPS][AR_STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk, kvh = blockIdx.z;
    if (warp == 0) {
        const Sequence f = find_block<false>(a, blockIdx.x, G, AR_ROWS);
        if (lane == 0) s_seq = f;
    }
    __syncthreads();
    const Sequence sq = s_seq;
    if (sq.b < 0) return;
    const int r0 = sq.blk * AR_ROWS, nrows = min(AR_ROWS, sq.nq * G - r0);
    const int off = sq.nk - sq.nq;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const KeyTiles kt = key_tiles(r0 / G + off, (r0 + nrows - 1) / G + off, sq.nk, left, right, a.sinks, AR_KEYS);

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
    const uint32_t ring = smem_u32(sm) + warp * AR_STAGES * STAGE;
    const int workers = plan.splits * AR_WARPS, me = blockIdx.y * AR_WARPS + warp;
    const T* kbase = static_cast<const T*>(a.k) + static_cast<int64_t>(sq.k0) * a.k_stride_t + kvh * a.k_stride_h;
    const T* vbase = static_cast<const T*>(a.v) + static_cast<int64_t>(sq.k0) * a.v_stride_t + kvh * a.v_stride_h;

    auto kept = [&](int t) -> bool {                     // this lane's key of tile index t may be seen
        if (t >= kt.count) return false;
        const int j = kt.tile(t) * AR_KEYS + lane;
        return j < sq.nk && (a.keep == nullptr || a.keep[sq.k0 + j] != 0);
    };
    bool next_kept = kept(me);
    auto issue = [&](int t, int stage) {
        const uint32_t word = __ballot_sync(0xffffffffu, next_kept);
        next_kept = kept(t + workers);
        if (t < kt.count) {
            const int j0 = kt.tile(t) * AR_KEYS;
            const uint32_t base = ring + stage * STAGE;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int idx = k * 32 + lane, r = idx / CH, c = idx % CH;
                const bool live = ((word >> r) & 1u) && c * 8 < a.D;
                const uint32_t dst = base + r * (DP * 2) + ((c ^ (r & 7)) << 4);
                const int64_t j = live ? j0 + r : 0;
                const int cc = live ? c * 8 : 0;
                cp16(dst, kbase + j * a.k_stride_t + cc, live);
                cp16(dst + AR_KEYS * DP * 2, vbase + j * a.v_stride_t + cc, live);
            }
            if (lane == 0) s_words[warp][stage] = word;
        }
        cp_commit();
    };

    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const float sc = a.scale * ATT_LOG2E;
    int issued = me, stage = 0;
#pragma unroll
    for (int k = 0; k < AR_STAGES - 1; ++k) {
        issue(issued, k);
        issued += workers;
    }
    for (int t = me; t < kt.count; t += workers) {
        cp_wait<AR_STAGES - 2>();
        __syncwarp();
        const uint32_t kb = ring + stage * STAGE, vb = kb + AR_KEYS * DP * 2;
        const uint32_t word = s_words[warp][stage];
        float s[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
        const int mat = lane >> 3, mr = lane & 7;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int np = 0; np < 2; ++np) {
                uint32_t b[4];
                const int key = np * 16 + (mat >> 1) * 8 + mr, ch = kk * 2 + (mat & 1);
                ldsm4(b, kb + key * (DP * 2) + ((ch ^ (key & 7)) << 4));
                mma16<T>(s[2 * np], qf[kk], b[0], b[1]);
                mma16<T>(s[2 * np + 1], qf[kk], b[2], b[3]);
            }
        const int j0 = kt.tile(t) * AR_KEYS;
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int jl = n * 8 + (lane & 3) * 2 + (e & 1), j = j0 + jl, p = pos[e >> 1];
                const bool see = ((word >> jl) & 1u) && j <= p + right && (j >= p - left || j < a.sinks);
                s[n][e] = see ? s[n][e] * sc : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
        float mref[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            mref[h] = mx[h] == -INFINITY ? 0.0f : mx[h];       // a row that has seen nothing yet
            const float f = exp2f(m[h] - mref[h]);
            m[h] = mx[h];
            l[h] *= f;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
                o[n][2 * h] *= f;
                o[n][2 * h + 1] *= f;
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = exp2f(s[n][e] - mref[e >> 1]);
                l[e >> 1] += s[n][e];
            }
#pragma unroll
        for (int kp = 0; kp < 2; ++kp) {
            // weights in [0, 1] rounded to the values' type, the type of the matrix instruction
            const uint32_t p[4] = {pack2(T(), s[2 * kp][0], s[2 * kp][1]), pack2(T(), s[2 * kp][2], s[2 * kp][3]),
                                   pack2(T(), s[2 * kp + 1][0], s[2 * kp + 1][1]),
                                   pack2(T(), s[2 * kp + 1][2], s[2 * kp + 1][3])};
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                const int key = kp * 16 + (mat & 1) * 8 + mr, ch = n * 2 + (mat >> 1);
                ldsm4t(b, vb + key * (DP * 2) + ((ch ^ (key & 7)) << 4));
                mma16<T>(o[2 * n], p, b[0], b[1]);
                mma16<T>(o[2 * n + 1], p, b[2], b[3]);
            }
        }
        __syncwarp();                                    // every lane has read the stage
        int fill = stage + AR_STAGES - 1;
        if (fill >= AR_STAGES) fill -= AR_STAGES;
        issue(issued, fill);
        issued += workers;
        if (++stage == AR_STAGES) stage = 0;
    }
    cp_wait<0>();
    __syncthreads();                                     // the rings are free: join the warps there
    float* so = reinterpret_cast<float*>(sm);            // [warp][16][DP]
    float* sml = so + AR_WARPS * AR_ROWS * DP;           // [warp][16][2]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = lane / 4 + 8 * h;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                so[(warp * AR_ROWS + r) * DP + n * 8 + (lane & 3) * 2 + e] = o[n][2 * h + e];
        if ((lane & 3) == 0) {
            sml[(warp * AR_ROWS + r) * 2] = m[h];
            sml[(warp * AR_ROWS + r) * 2 + 1] = l[h];
        }
    }
    __syncthreads();
    const size_t slot = (static_cast<size_t>(blockIdx.x) * a.Hk + kvh) * plan.splits + blockIdx.y;
    for (int k = threadIdx.x; k < nrows * DP; k += AR_WARPS * 32) {
        const int r = k / DP, d = k % DP;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < AR_WARPS; ++w) mm = fmaxf(mm, sml[(w * AR_ROWS + r) * 2]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ov = 0.0f, lv = 0.0f;
#pragma unroll
        for (int w = 0; w < AR_WARPS; ++w) {
            const float f = exp2f(sml[(w * AR_ROWS + r) * 2] - ref);
            ov = fmaf(f, so[(w * AR_ROWS + r) * DP + d], ov);
            lv = fmaf(f, sml[(w * AR_ROWS + r) * 2 + 1], lv);
        }
        if (plan.splits > 1) {
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

// Adds the shares of a row block: weights 2^(m_s - max m).
template <typename T, int DP>
__global__ void __launch_bounds__(128) attn_join_kernel(const dn8_attention_args a, const RowsPlan plan) {
    __shared__ Sequence s_seq;
    const int G = a.Hq / a.Hk, kvh = blockIdx.y;
    if (threadIdx.x < 32) {
        const Sequence f = find_block<false>(a, blockIdx.x, G, AR_ROWS);
        if (threadIdx.x == 0) s_seq = f;
    }
    __syncthreads();
    const Sequence sq = s_seq;
    if (sq.b < 0) return;
    const int r0 = sq.blk * AR_ROWS, nrows = min(AR_ROWS, sq.nq * G - r0);
    const size_t slot = (static_cast<size_t>(blockIdx.x) * a.Hk + kvh) * plan.splits;
    griddep_wait();
    for (int k = threadIdx.x; k < nrows * DP; k += 128) {
        const int r = k / DP, d = k % DP;
        float mm = -INFINITY;
        for (int s = 0; s < plan.splits; ++s) mm = fmaxf(mm, plan.ml[((slot + s) * AR_ROWS + r) * 2]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ov = 0.0f, lv = 0.0f;
        for (int s = 0; s < plan.splits; ++s) {
            const float* ml = plan.ml + ((slot + s) * AR_ROWS + r) * 2;
            const float f = exp2f(ml[0] - ref);
            ov = fmaf(f, plan.o[((slot + s) * AR_ROWS + r) * DP + d], ov);
            lv = fmaf(f, ml[1], lv);
        }
        const int64_t row = sq.q0 + (r0 + r) / G;
        const int h = kvh * G + (r0 + r) % G;
        if (d < a.D)
            (static_cast<T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h)[d] = from_f32<T>(lv > 0.0f ? ov / lv : 0.0f);
        if (d == 0 && a.lse != nullptr) a.lse[row * a.Hq + h] = lv > 0.0f ? (mm + log2f(lv)) * ATT_LN2 : -INFINITY;
    }
}

namespace {

int head_pad(int D) { return D <= 64 ? 64 : 128; }

// Row blocks (a bound: every sequence may leave one block unfilled) and shares of the key axis: as many
// as give every SM a few CTAs while a warp still has a handful of tiles of an average sequence.
RowsPlan rows_plan(const dn8_attention_args& a, int sms) {
    RowsPlan p = {};
    const int64_t rows = a.Tq * (a.Hq / a.Hk);
    p.blocks = static_cast<int>(rows / AR_ROWS + (a.B < rows ? a.B : rows));
    int64_t seen = a.Tk / a.B;
    if (a.left >= 0 && a.right >= 0) {
        const int64_t w = static_cast<int64_t>(a.left) + a.right + 1 + a.sinks + a.Tq / a.B;
        if (w < seen) seen = w;
    }
    const int64_t tiles = (seen + AR_KEYS - 1) / AR_KEYS;
    int64_t s = 8ll * sms / (static_cast<int64_t>(p.blocks) * a.Hk);
    if (s > tiles / (4 * AR_WARPS)) s = tiles / (4 * AR_WARPS);
    p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
    return p;
}
size_t rows_work(const dn8_attention_args& a, const RowsPlan& p) {
    if (p.splits == 1) return 0;
    return static_cast<size_t>(p.blocks) * a.Hk * p.splits * AR_ROWS * (head_pad(a.D) + 2) * sizeof(float);
}

template <typename T, int DP> cudaError_t rows_go(const dn8_attention_args& a, RowsPlan p, cudaStream_t st) {
    const size_t ring = static_cast<size_t>(AR_WARPS) * AR_STAGES * 2 * AR_KEYS * DP * 2;
    const size_t join = static_cast<size_t>(AR_WARPS) * AR_ROWS * (DP + 2) * 4;
    const size_t smem = ring > join ? ring : join;
    cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (p.splits > 1) {
        p.o = static_cast<float*>(a.work);
        p.ml = p.o + static_cast<size_t>(p.blocks) * a.Hk * p.splits * AR_ROWS * DP;
    }
    e = launch_pdl(false, attn_rows_kernel<T, DP>, dim3(p.blocks, p.splits, a.Hk), dim3(AR_WARPS * 32), smem, st, a, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_pdl(true, attn_join_kernel<T, DP>, dim3(p.blocks, a.Hk), dim3(128), 0, st, a, p);
}

}  // namespace

// Few rows per sequence and key head: the row kernel, which packs the heads of a group and splits the
// key axis. Otherwise 128-row tiles on the tensor cores (attn_tile.cu).
static bool few_rows(const dn8_attention_args& a) { return a.Tq * (a.Hq / a.Hk) <= 32ll * a.B; }

size_t attention_work(const dn8_attention_args& a, int sms) { return few_rows(a) ? rows_work(a, rows_plan(a, sms)) : 0; }

cudaError_t launch_attention(const dn8_attention_args& a, int sms, cudaStream_t st) {
    if (!few_rows(a)) return launch_attention_tile(a, st);
    const RowsPlan p = rows_plan(a, sms);
    if (a.type == DN8_F16) return head_pad(a.D) == 64 ? rows_go<__half, 64>(a, p, st) : rows_go<__half, 128>(a, p, st);
    return head_pad(a.D) == 64 ? rows_go<__nv_bfloat16, 64>(a, p, st) : rows_go<__nv_bfloat16, 128>(a, p, st);
}

}  // namespace dn8
