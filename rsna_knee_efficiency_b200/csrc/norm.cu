// norm.cu -- layer norm over the rows of a matrix, forward and backward, with the residual sum in
// front of it and the reduction of the weight's and the bias's gradient.
//
//   h = x + res (rounded to x's type: the stored sum is what the statistics, and later the backward
//   pass, see), mu = sum h / C, var = sum (h - mu)^2 / C, r = 1 / sqrt(var + eps), y = (h - mu) r w + b
//   g = dy w, xh = (h - mu) r, dx = r (g - mean(g) - xh mean(g xh)) + dsum, dw = sum dy xh, db = sum dy
//
// Both passes are bound by memory: a row is read once into registers (a team of 8, 32, 128 or 512
// threads per row, so that a thread holds at most 32 values), the variance is summed from the
// registers as squares of differences (no cancellation of E[x^2] - mu^2), and written once.
// Statistics and sums are fp32. 98304 rows of 512 bf16 with a residual (403 MB): 77 us, 5.2 TB/s of 6.5 for a copy.
// Narrow rows share a warp: 67678 rows of 31 bf16 took 52 us with a warp each and
// take 11 with eight threads each, 90000 of 64 (fp32 in, fp16 out) 40 and 17.
#include "ctx_common.cuh"
#include "dn8_kernels.h"

namespace dn8 {

// Sums of values per thread over a team of TPR threads; every thread gets the same ones. `red`, a float per value
// and warp, is the team's, and free once the team has passed another barrier: two calls in a row use two of them.
// (One barrier per sum, of the team alone, not two of the block: 27056 rows of 1848 fp32 with a residual 136 -> 120 us.)
// Teams of less than a warp do not wait for one another.
template <int TPR> DN8_DEV float lanes_sum(float v) {
    if (TPR >= 32) return warp_sum(v);
    const uint32_t mask = ((1u << (TPR % 32)) - 1u) << (threadIdx.x & 31 & ~(TPR - 1));
#pragma unroll
    for (int k = TPR / 2; k > 0; k >>= 1) v += __shfl_xor_sync(mask, v, k);
    return v;
}
template <int TPR> DN8_DEV void team_barrier() {
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / TPR), "n"(TPR < 32 ? 32 : TPR) : "memory");
}
template <int TPR> DN8_DEV float team_sum(float v, float* red) {
    v = lanes_sum<TPR>(v);
    if (TPR <= 32) return v;
    const int warp = (threadIdx.x % TPR) >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    team_barrier<TPR>();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) s += red[w];
    return s;
}
template <int TPR> DN8_DEV void team_sum2(float& a, float& b, float* red) {
    a = lanes_sum<TPR>(a);
    b = lanes_sum<TPR>(b);
    if (TPR <= 32) return;
    const int warp = (threadIdx.x % TPR) >> 5;
    if ((threadIdx.x & 31) == 0) {
        red[warp] = a;
        red[TPR / 32 + warp] = b;
    }
    team_barrier<TPR>();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) {
        a += red[w];
        b += red[TPR / 32 + w];
    }
}

// A team's rows are gridDim.x teams apart; the next row's loads are in flight while this one is reduced.
// Weight and bias, for every row of a team the same, come from shared memory: in registers they cost
// more in warps per SM than they save, and warps are what keeps enough bytes in flight.
template <typename TX, typename TY, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, TPR < 512 ? (VEC * NV <= 16 ? 8 : 4) : (VEC * NV <= 16 ? 2 : 1))
ln_kernel(const dn8_layer_norm_args a) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, TEAMS = THREADS / TPR;
    __shared__ float red[2][TPR < 32 ? 1 : TPR / 32];
    extern __shared__ __align__(16) float wb[];              // [C] weights, [C] biases
    const int t = threadIdx.x % TPR, C = a.C;
    const int64_t step = static_cast<int64_t>(gridDim.x) * TEAMS;
    int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + threadIdx.x / TPR;
    Vec<TX, VEC> nx[NV], nr[NV];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (t + k * TPR) * VEC;
            if (c < C) {
                nx[k] = load_vec<TX, VEC>(static_cast<const TX*>(a.x) + r * a.x_stride + c);
                if (a.res != nullptr)
                    nr[k] = load_vec<TX, VEC>(static_cast<const TX*>(a.res) + r * a.res_stride + c);
            }
        }
    };
    if (row < a.rows) fetch(row);
    for (int c = threadIdx.x * VEC; c < C; c += THREADS * VEC) {
        float w[VEC], bi[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            w[e] = 1.0f;
            bi[e] = 0.0f;
        }
        if (a.w != nullptr) load_param(a.w, a.w_type, c, w);
        if (a.b != nullptr) load_param(a.b, a.w_type, c, bi);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            wb[c + e] = w[e];
            wb[C + c + e] = bi[e];
        }
    }
    __syncthreads();
    if (row >= a.rows) return;                               // a whole team (TPR > 32: a whole block)
    for (; row < a.rows; row += step) {
        float h[NV][VEC];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (t + k * TPR) * VEC;
            if (c < C) {
                if (a.res != nullptr) {
                    Vec<TX, VEC> s;
                    float rv[VEC];
                    nx[k].get(h[k]);
                    nr[k].get(rv);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) h[k][e] += rv[e];
                    s.set(h[k]);
                    store_vec(static_cast<TX*>(a.sum) + row * a.sum_stride + c, s);
                    s.get(h[k]);
                } else {
                    nx[k].get(h[k]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[k][e] = 0.0f;
            }
        }
        if (row + step < a.rows) fetch(row + step);
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += h[k][e];
        const float mu = team_sum<TPR>(s, red[0]) / static_cast<float>(C);
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if ((t + k * TPR) * VEC < C)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    h[k][e] -= mu;
                    q = fmaf(h[k][e], h[k][e], q);
                }
        const float r = rsqrtf(team_sum<TPR>(q, red[1]) / static_cast<float>(C) + a.eps);
        TY* y = static_cast<TY*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (t + k * TPR) * VEC;
            if (c < C) {
                float o[VEC], w[VEC], bi[VEC];
                load_f32(wb + c, w);
                load_f32(wb + C + c, bi);
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = fmaf(h[k][e] * r, w[e], bi[e]);
                store_f32(y + c, o);
            }
        }
        if (t == 0) {
            if (a.mean != nullptr) a.mean[row] = mu;
            if (a.rstd != nullptr) a.rstd[row] = r;
        }
    }
}

// Rows longer than a team's registers hold: one block per row, the sum's row read again (from L2) for
// the variance and for the output.
template <typename TX, typename TY>
__global__ void __launch_bounds__(512) ln_long_kernel(const dn8_layer_norm_args a) {
    __shared__ float red[2][16];
    const int64_t row = blockIdx.x;
    const int C = a.C;
    const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
    TX* sum = a.res != nullptr ? static_cast<TX*>(a.sum) + row * a.sum_stride : nullptr;
    const TX* res = a.res != nullptr ? static_cast<const TX*>(a.res) + row * a.res_stride : nullptr;
    float s = 0.0f;
    for (int c = threadIdx.x; c < C; c += 512) {
        float v = to_f32(x[c]);
        if (res != nullptr) {
            const TX hv = from_f32<TX>(v + to_f32(res[c]));
            sum[c] = hv;
            v = to_f32(hv);
        }
        s += v;
    }
    const TX* h = res != nullptr ? sum : x;                  // a thread reads back its own columns
    const float mu = team_sum<512>(s, red[0]) / static_cast<float>(C);
    float q = 0.0f;
    for (int c = threadIdx.x; c < C; c += 512) {
        const float d = to_f32(h[c]) - mu;
        q = fmaf(d, d, q);
    }
    const float r = rsqrtf(team_sum<512>(q, red[1]) / static_cast<float>(C) + a.eps);
    TY* y = static_cast<TY*>(a.y) + row * a.y_stride;
    for (int c = threadIdx.x; c < C; c += 512) {
        float w[1] = {1.0f}, b[1] = {0.0f};
        if (a.w != nullptr) load_param(a.w, a.w_type, c, w);
        if (a.b != nullptr) load_param(a.b, a.w_type, c, b);
        y[c] = from_f32<TY>(fmaf((to_f32(h[c]) - mu) * r, w[0], b[0]));
    }
    if (threadIdx.x == 0) {
        if (a.mean != nullptr) a.mean[row] = mu;
        if (a.rstd != nullptr) a.rstd[row] = r;
    }
}

// BYTES from global to shared memory, asynchronously; wait_copies: all but the `n` last committed groups have come.
template <int BYTES> DN8_DEV void copy_async(void* dst, const void* src) {
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
DN8_DEV void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
DN8_DEV void wait_copies(int n) {
    if (n >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (n >= 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Backward: persistent blocks of TEAMS teams; a thread keeps the same columns for every row, so the sums of dy xh
// and dy over the block's rows stay in its registers. Rows of 16-byte vectors come through a ring of `stages` rows
// per team in shared memory: every thread copies and reads its own vectors, so nobody waits for anybody. (One
// row ahead in registers is too little in flight: 23664 rows of 2016, fp32 and fp16, took 117 us and take 88; 98304 of
// 512 bf16 with dsum 77 and 74, 5.4 TB/s; 20427 of 1064 fp16, bound by instructions, 50 and 53.) The sums are added
// over the teams in shared memory and written as one row of the workspace [gridDim.x][2][C]; ln_cols_kernel adds
// the rows in a fixed order (no atomics: the same bits every call).
template <typename TX, typename TY, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR < 512 ? 2 : 1) ln_bwd_kernel(const dn8_layer_norm_bwd_args a,
                                                                                                       int stages) {
    constexpr int THREADS = TPR < 256 ? 256 : TPR;
    constexpr int TEAMS = THREADS / TPR, CB = NV * VEC * TPR;      // columns a team covers
    __shared__ float red[TEAMS][2][TPR < 32 ? 1 : 2 * TPR / 32];
    __shared__ float part[TEAMS > 1 ? 2 * CB : 1];
    griddep_launch_dependents();
    extern __shared__ __align__(16) float ws_[];             // [C] weights, then the ring
    const int team = threadIdx.x / TPR, t = threadIdx.x % TPR, C = a.C;
    float dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.0f;
    for (int c = threadIdx.x * VEC; c < C; c += THREADS * VEC) {
        float w[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] = 1.0f;
        if (a.w != nullptr) load_param(a.w, a.w_type, c, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ws_[c + e] = w[e];
    }
    __syncthreads();
    const float inv_c = 1.0f / static_cast<float>(C);
    // (every team of a block makes the same number of steps)
    const int64_t step = static_cast<int64_t>(gridDim.x) * TEAMS;
    constexpr bool RING = VEC > 1;
    constexpr int SX = VEC * sizeof(TX), SY = VEC * sizeof(TY);
    Vec<TX, VEC> nx[NV], nd[NV];
    Vec<TY, VEC> ng[NV];
    float nmu = 0.0f, nr = 0.0f;                             // mean and rstd: one row ahead
    auto fetch_stats = [&](int64_t r) {
        if (r >= a.rows) return;
        nmu = a.mean[r];
        nr = a.rstd[r];
    };
    // a team's row in the ring: x, dy, dsum
    const int row_bytes = C * static_cast<int>(2 * sizeof(TX) + sizeof(TY));
    uint8_t* ring = reinterpret_cast<uint8_t*>(ws_ + C) + static_cast<size_t>(team) * stages * row_bytes;
    auto fetch = [&](int64_t r, int stage) {
        if (r < a.rows) {
            uint8_t* slot = ring + stage * row_bytes;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (t + k * TPR) * VEC;
                if (c < C) {
                    const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride + c;
                    const TY* dy = static_cast<const TY*>(a.dy) + r * a.dy_stride + c;
                    const TX* ds = a.dsum != nullptr ? static_cast<const TX*>(a.dsum) + r * a.dsum_stride + c : nullptr;
                    if constexpr (RING) {
                        copy_async<SX>(slot + c * sizeof(TX), x);
                        copy_async<SY>(slot + C * sizeof(TX) + c * sizeof(TY), dy);
                        if (ds != nullptr) copy_async<SX>(slot + C * (sizeof(TX) + sizeof(TY)) + c * sizeof(TX), ds);
                    } else {
                        nx[k] = load_vec<TX, VEC>(x);
                        ng[k] = load_vec<TY, VEC>(dy);
                        if (ds != nullptr) nd[k] = load_vec<TX, VEC>(ds);
                    }
                }
            }
        }
        if (RING) commit_copies();
    };
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
    for (int s = 0; s < stages; ++s) fetch(row0 + s * step, s);
    fetch_stats(row0);
    int stage = 0, odd = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * TEAMS; base < a.rows; base += step) {
        const int64_t row = base + team;
        const bool live = row < a.rows;
        float dy[NV][VEC], xh[NV][VEC];
        Vec<TX, VEC> d[NV];
        float s1 = 0.0f, s2 = 0.0f;
        const float mu = nmu, r = nr;
        fetch_stats(row + step);
        if (RING) wait_copies(stages - 1);
        if (live) {
            const uint8_t* slot = ring + stage * row_bytes;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if ((t + k * TPR) * VEC < C) {
                    float w[VEC];
                    load_f32(ws_ + (t + k * TPR) * VEC, w);
                    if (RING) {
                        const int c = (t + k * TPR) * VEC;
                        nx[k] = *reinterpret_cast<const Vec<TX, VEC>*>(slot + c * sizeof(TX));
                        ng[k] = *reinterpret_cast<const Vec<TY, VEC>*>(slot + C * sizeof(TX) + c * sizeof(TY));
                        if (a.dsum != nullptr)
                            nd[k] = *reinterpret_cast<const Vec<TX, VEC>*>(slot + C * (sizeof(TX) + sizeof(TY)) + c * sizeof(TX));
                    }
                    d[k] = nd[k];
                    nx[k].get(xh[k]);
                    ng[k].get(dy[k]);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        xh[k][e] = (xh[k][e] - mu) * r;
                        dw[k][e] = fmaf(dy[k][e], xh[k][e], dw[k][e]);
                        db[k][e] += dy[k][e];
                        dy[k][e] *= w[e];
                        s1 += dy[k][e];
                        s2 = fmaf(dy[k][e], xh[k][e], s2);
                    }
                }
        }
        fetch(row + stages * step, stage);
        if (++stage == stages) stage = 0;
        team_sum2<TPR>(s1, s2, red[team][odd]);
        odd ^= 1;
        if (!live) continue;
        s1 *= inv_c;
        s2 *= inv_c;
        TX* dx = static_cast<TX*>(a.dx) + row * a.dx_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (t + k * TPR) * VEC;
            if (c < C) {
                float o[VEC], dv[VEC] = {};
                if (a.dsum != nullptr) d[k].get(dv);
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = r * (dy[k][e] - s1 - xh[k][e] * s2) + dv[e];
                store_f32(dx + c, o);
            }
        }
    }
    if (a.work == nullptr) return;
    float* ws = static_cast<float*>(a.work) + static_cast<size_t>(blockIdx.x) * 2 * C;
    if (TEAMS > 1) {
        // one team after the other adds its sums (a fixed order)
        for (int m = 0; m < TEAMS; ++m) {
            if (team == m)
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int c = (t + k * TPR) * VEC + e;
                        part[c] = (m ? part[c] : 0.0f) + dw[k][e];
                        part[CB + c] = (m ? part[CB + c] : 0.0f) + db[k][e];
                    }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < C; c += THREADS) {
            ws[c] = part[c];
            ws[C + c] = part[CB + c];
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int c = (t + k * TPR) * VEC + e;
                if (c < C) {
                    ws[c] = dw[k][e];
                    ws[C + c] = db[k][e];
                }
            }
    }
}

// Rows longer than a team's registers hold: dx by one block per row (dy and h read twice) ...
template <typename TX, typename TY>
__global__ void __launch_bounds__(512) ln_bwd_long_kernel(const dn8_layer_norm_bwd_args a) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const int C = a.C;
    const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
    const TY* dy = static_cast<const TY*>(a.dy) + row * a.dy_stride;
    const float mu = a.mean[row], r = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < C; c += 512) {
        float w[1] = {1.0f};
        if (a.w != nullptr) load_param(a.w, a.w_type, c, w);
        const float g = to_f32(dy[c]) * w[0];
        s1 += g;
        s2 = fmaf(g, (to_f32(x[c]) - mu) * r, s2);
    }
    team_sum2<512>(s1, s2, red);
    s1 /= static_cast<float>(C);
    s2 /= static_cast<float>(C);
    TX* dx = static_cast<TX*>(a.dx) + row * a.dx_stride;
    for (int c = threadIdx.x; c < C; c += 512) {
        float w[1] = {1.0f};
        if (a.w != nullptr) load_param(a.w, a.w_type, c, w);
        float o = r * (to_f32(dy[c]) * w[0] - s1 - (to_f32(x[c]) - mu) * r * s2);
        if (a.dsum != nullptr) o += to_f32((static_cast<const TX*>(a.dsum) + row * a.dsum_stride)[c]);
        dx[c] = from_f32<TX>(o);
    }
}
// ... and the sums of a slab of rows (blockIdx.y of gridDim.y) by one thread per column. It runs before
// ln_bwd_long_kernel, whose dx may be dy's or dsum's own memory.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256) ln_bwd_long_cols_kernel(const dn8_layer_norm_bwd_args a) {
    const int c = blockIdx.x * 256 + threadIdx.x, C = a.C;
    if (c >= C) return;
    const int64_t per = (a.rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = per * blockIdx.y, r1 = min(a.rows, r0 + per);
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = r0; row < r1; ++row) {
        const float dy = to_f32(static_cast<const TY*>(a.dy)[row * a.dy_stride + c]);
        const float h = to_f32(static_cast<const TX*>(a.x)[row * a.x_stride + c]);
        dw = fmaf(dy, (h - a.mean[row]) * a.rstd[row], dw);
        db += dy;
    }
    float* ws = static_cast<float*>(a.work) + static_cast<size_t>(blockIdx.y) * 2 * C;
    ws[c] = dw;
    ws[C + c] = db;
}

// dw, db = the sum of the workspace's rows: 32 columns per block, 32 threads adding every 32nd row of
// a column, then a fixed tree.
__global__ void __launch_bounds__(1024) ln_cols_kernel(const float* work, int nrows, int C, void* dw, void* db, int type) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;                    // column of [2][C]
    griddep_wait();
    float s = 0.0f;
    if (c < 2 * C)
        for (int r = ty; r < nrows; r += 32) s += work[static_cast<size_t>(r) * 2 * C + c];
    part[ty][lane] = s;
    __syncthreads();
    s = warp_sum(part[lane][ty]);                            // column ty of the block's 32
    const int co = blockIdx.x * 32 + ty;
    if (lane == 0 && co < 2 * C) {
        void* dst = co < C ? dw : db;
        const int k = co < C ? co : co - C;
        if (dst == nullptr) return;
        if (type == DN8_F32) static_cast<float*>(dst)[k] = s;
        else if (type == DN8_F16) static_cast<__half*>(dst)[k] = __float2half_rn(s);
        else static_cast<__nv_bfloat16*>(dst)[k] = __float2bfloat16_rn(s);
    }
}

namespace {

bool vec_ok(const void* p, int64_t stride, int size) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride * size) % 16 == 0;
}
int type_size(int type) { return type == DN8_F32 ? 4 : 2; }

constexpr int LN_COLS_ROWS = 296;       // rows of the backward pass's workspace (two blocks per SM)

// x's and y's types: equal, or fp32 in and 16 bits out
template <typename F> cudaError_t with_types(int tx, int ty, F&& f) {
    if (tx == ty) return with_type(tx, [&](auto t) { return f(t, t); });
    if (tx != DN8_F32) return cudaErrorInvalidValue;
    return ty == DN8_F16 ? f(float(), __half()) : f(float(), __nv_bfloat16());
}

// Blocks: enough for every SM's threads (8 blocks of 128 threads hold the registers of an SM), each with
// several rows per team when there are many.
template <typename TX, typename TY, int VEC, int NV, int TPR>
cudaError_t ln_team(const dn8_layer_norm_args& a, int sms, cudaStream_t st) {
    constexpr int THREADS = TPR < 128 ? 128 : TPR, TEAMS = THREADS / TPR;
    const int64_t want = (a.rows + TEAMS - 1) / TEAMS, most = static_cast<int64_t>(sms) * (1024 / THREADS);
    const size_t smem = static_cast<size_t>(a.C) * 2 * sizeof(float);
    if (smem > 40 * 1024) {
        // (the most that any call of this instance asks for, not this call's own: another host thread with a
        // narrower row may set the limit between here and the launch)
        cudaError_t e = cudaFuncSetAttribute(ln_kernel<TX, TY, VEC, NV, TPR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             VEC * NV * TPR * 2 * static_cast<int>(sizeof(float)));
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(false, ln_kernel<TX, TY, VEC, NV, TPR>, dim3(static_cast<unsigned>(want < most ? want : most)),
                      dim3(THREADS), smem, st, a);
}
// The smallest team that holds a row: 16 elements per thread, else up to 32 (and then 16 in wider teams)
template <typename TX, typename TY, int VEC, int NV>
cudaError_t ln_go(const dn8_layer_norm_args& a, int sms, cudaStream_t st) {
    constexpr int per = VEC * NV;
    if (a.C <= 8 * per) return ln_team<TX, TY, VEC, NV, 8>(a, sms, st);
    if (a.C <= 32 * per) return ln_team<TX, TY, VEC, NV, 32>(a, sms, st);
    // (more single elements per thread keep too few warps at work)
    if (VEC > 1 && a.C <= 64 * per) return ln_team<TX, TY, VEC, 2 * NV, 32>(a, sms, st);
    if (a.C <= 128 * per) return ln_team<TX, TY, VEC, NV, 128>(a, sms, st);
    if (VEC > 1 && a.C <= 256 * per) return ln_team<TX, TY, VEC, 2 * NV, 128>(a, sms, st);
    if (a.C <= 512 * per) return ln_team<TX, TY, VEC, NV, 512>(a, sms, st);
    if (a.C <= 1024 * per) return ln_team<TX, TY, VEC, 2 * NV, 512>(a, sms, st);
    return launch_pdl(false, ln_long_kernel<TX, TY>, dim3(static_cast<unsigned>(a.rows)), dim3(512), 0, st, a);
}

template <typename TX, typename TY, int VEC, int NV>
cudaError_t ln_bwd_go(const dn8_layer_norm_bwd_args& a, cudaStream_t st, int* nrows) {
    const int per = VEC * NV;
    const int teams = a.C <= 8 * per ? 32 : a.C <= 32 * per ? 8 : a.C <= 128 * per ? 2 : 1;
    const int64_t want = (a.rows + teams - 1) / teams;
    const int grid = static_cast<int>(want < LN_COLS_ROWS ? want : LN_COLS_ROWS);
    *nrows = grid;
    if (a.C <= 512 * per) {
        // Stages: four rows per team, two or one where they would not leave room for two blocks per SM (teams of
        // 512: for one)
        const size_t most = a.C <= 128 * per ? 80 * 1024 : 180 * 1024;
        const size_t rows = static_cast<size_t>(teams) * a.C * (2 * sizeof(TX) + sizeof(TY));
        const int stages = VEC == 1 ? 1 : 4 * rows <= most ? 4 : 2 * rows <= most ? 2 : 1;
        const size_t smem = static_cast<size_t>(a.C) * sizeof(float) + (VEC == 1 ? 0 : stages * rows);
        const auto kernel = a.C <= 8 * per     ? ln_bwd_kernel<TX, TY, VEC, NV, 8>
                            : a.C <= 32 * per  ? ln_bwd_kernel<TX, TY, VEC, NV, 32>
                            : a.C <= 128 * per ? ln_bwd_kernel<TX, TY, VEC, NV, 128>
                                               : ln_bwd_kernel<TX, TY, VEC, NV, 512>;
        // (the default limit of 48 KB counts the static part too: up to 16.5 KB, the sums of teams of 128)
        if (smem > 24 * 1024) {
            // (as in ln_team: the most that any call of the instance asks for)
            const size_t cols = static_cast<size_t>(per) * (a.C <= 8 * per ? 8 : a.C <= 32 * per ? 32 : a.C <= 128 * per ? 128 : 512);
            const size_t widest = teams * cols * (2 * sizeof(TX) + sizeof(TY));
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(cols * sizeof(float) + (widest > most ? widest : most)));
            if (e != cudaSuccess) return e;
        }
        return launch_pdl(false, kernel, dim3(grid), dim3(a.C <= 128 * per ? 256 : 512), smem, st, a, stages);
    }
    if (a.work != nullptr) {
        const int slabs = static_cast<int>(a.rows < 32 ? 1 : a.rows / 32 < LN_COLS_ROWS ? a.rows / 32 : LN_COLS_ROWS);
        *nrows = slabs;
        cudaError_t e = launch_pdl(false, ln_bwd_long_cols_kernel<TX, TY>, dim3((a.C + 255) / 256, slabs), dim3(256), 0, st, a);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(false, ln_bwd_long_kernel<TX, TY>, dim3(static_cast<unsigned>(a.rows)), dim3(512), 0, st, a);
}

}  // namespace

cudaError_t launch_layer_norm(const dn8_layer_norm_args& a, int sms, cudaStream_t st) {
    const int sx = type_size(a.x_type), sy = type_size(a.y_type);
    const bool vec = a.C % 8 == 0 && vec_ok(a.w, 0, 4) && vec_ok(a.b, 0, 4) && vec_ok(a.x, a.x_stride, sx) &&
                     vec_ok(a.y, a.y_stride, sy) &&
                     (a.res == nullptr || (vec_ok(a.res, a.res_stride, sx) && vec_ok(a.sum, a.sum_stride, sx)));
    // two elements of every row (and of weight and bias) at a time
    auto pairs_of = [](const void* p, int64_t stride, int size) {
        return reinterpret_cast<uintptr_t>(p) % (2 * size) == 0 && stride % 2 == 0;
    };
    const bool two = a.C % 2 == 0 && pairs_of(a.w, 0, 4) && pairs_of(a.b, 0, 4) && pairs_of(a.x, a.x_stride, sx) &&
                     pairs_of(a.y, a.y_stride, sy) &&
                     (a.res == nullptr || (pairs_of(a.res, a.res_stride, sx) && pairs_of(a.sum, a.sum_stride, sx)));
    return with_types(a.x_type, a.y_type, [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        // 16-byte loads where every row allows them, pairs where C is even (40000 rows of 514 bf16 with a residual:
        // 45 us, 67 with half as many per thread; 8000 of 2050 fp32: 71, and 45), else single elements, eight per thread
        // (40000 rows of 515: 88 us; with sixteen, 189)
        if (!vec && two) return a.C <= 1024 ? ln_go<TX, TY, 2, 8>(a, sms, st) : ln_go<TX, TY, 2, 4>(a, sms, st);
        if (!vec) return ln_go<TX, TY, 1, 8>(a, sms, st);
        if constexpr (sizeof(TX) == 4) return ln_go<TX, TY, 4, 4>(a, sms, st);
        else return ln_go<TX, TY, 8, 2>(a, sms, st);
    });
}

size_t layer_norm_bwd_work(int C) { return static_cast<size_t>(LN_COLS_ROWS) * 2 * C * sizeof(float); }

cudaError_t launch_layer_norm_bwd(const dn8_layer_norm_bwd_args& args, cudaStream_t st) {
    dn8_layer_norm_bwd_args a = args;
    if (a.dw == nullptr && a.db == nullptr) a.work = nullptr;
    const int sx = type_size(a.x_type), sy = type_size(a.y_type);
    const bool vec = a.C % 8 == 0 && vec_ok(a.w, 0, 4) && vec_ok(a.x, a.x_stride, sx) && vec_ok(a.dy, a.dy_stride, sy) &&
                     vec_ok(a.dx, a.dx_stride, sx) && (a.dsum == nullptr || vec_ok(a.dsum, a.dsum_stride, sx));
    int nrows = 0;
    cudaError_t e = a.rows == 0 ? cudaSuccess : with_types(a.x_type, a.y_type, [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        if (!vec) return ln_bwd_go<TX, TY, 1, 8>(a, st, &nrows);
        if constexpr (sizeof(TX) == 4) return ln_bwd_go<TX, TY, 4, 4>(a, st, &nrows);
        else return ln_bwd_go<TX, TY, 8, 2>(a, st, &nrows);
    });
    if (e != cudaSuccess || a.work == nullptr) return e;
    return launch_pdl(nrows > 0, ln_cols_kernel, dim3((2 * a.C + 31) / 32), dim3(1024), 0, st,
                      static_cast<const float*>(a.work), nrows, a.C, a.dw, a.db, a.w_type);
}

}  // namespace dn8
