// rope.cu -- rotary positions with several axes (slot, slice, row, column, ...), applied to the queries
// and the keys of a sequence in one launch.
//
// The first 2 P elements of a head are P pairs, either (j, j + P) or (2 j, 2 j + 1); pair j belongs to
// one axis and turns by pos[token][axis(j)] f_j:  (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin).
// The backward pass is the turn by the negative angle. Elements behind the pairs are copied.
//
// Angles: a 32-bit product pos * f loses the fraction of a turn for far positions (pos = 10^6: 0.06
// rad), so f is kept in turns (f / 2 pi) as a double, the product is taken in 64 bits, its whole turns
// are dropped there and only the remaining fraction, within half a turn, goes on in 32 bits.
//
// Bound by memory (each element read and written once). A block holds the cos / sin of its tokens in
// shared memory, computed once per (token, pair), while its first items are on their way, and used by every head
// of q and k.
#include <cmath>

#include "ctx_common.cuh"
#include "dn8_kernels.h"

namespace dn8 {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_PAIRS = 128;
constexpr int RP_BATCH = 2;                       // items a thread has in flight
// Items of 16 bytes per thread that a block is cut for: 98304 tokens of 20 heads, D = 64, bf16 (503 MB): 99 us
// with 4, 93 with 8 (93 to 97 from one B200 to the next: 5.2 to 5.4 TB/s), 95 with 16; single elements (10626
// tokens, 10 heads, 31 pairs) 23, 29, 29.
constexpr int RP_BLOCK_WIDE = 8, RP_BLOCK_NARROW = 4;

struct RopeTable {
    double turns[RP_MAX_PAIRS];                   // f_j / (2 pi)
    uint8_t axis[RP_MAX_PAIRS];
};

// cs[t][j] of the block's tokens, `slots` per token (those behind the pairs: no turn). A thread keeps its pair for
// all its tokens: lanes that read different places of the table, which is a kernel argument, take turns (read
// for every token, 29497 tokens of 6 heads, D = 80, took 32 us, not 19).
DN8_DEV void turn_table(const dn8_rope_args& a, const RopeTable& tab, int pairs, int slots, int64_t t0, int nt, float2* cs) {
    const int rows = RP_THREADS / slots, j = threadIdx.x % slots;      // (slots <= RP_MAX_PAIRS)
    if (static_cast<int>(threadIdx.x) >= rows * slots) return;
    const bool live = j < pairs;
    const double turns = live ? tab.turns[j] : 0.0;
    const int axis = live ? tab.axis[j] : 0;
    for (int t = threadIdx.x / slots; t < nt; t += rows) {
        const double ang = static_cast<double>(a.pos[(t0 + t) * a.n_axes + axis]) * turns;
        const float fr = static_cast<float>(2.0 * (ang - rint(ang)));      // half turns in [-1, 1]
        float s, c;
        sincospif(fr, &s, &c);
        cs[t * slots + j] = make_float2(c, a.inverse ? -s : s);
    }
}

// Interleaved pairs, 16 bytes an item: D / VEC items per head, whatever the number of pairs (elements behind them
// are copied, not turned by nothing: 0 times an infinite neighbour is not 0).
template <typename T, int VEC>
__global__ void __launch_bounds__(RP_THREADS, 4) rope_inter_kernel(const dn8_rope_args a, const __grid_constant__ RopeTable tab,
                                                                   int pairs, int tokens_per_block) {
    constexpr int BATCH = 2 * RP_BATCH;
    extern __shared__ __align__(16) float2 cs[];  // [tokens of the block][slots]
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
    const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.T - t0));
    const int slots = (pairs + VEC / 2 - 1) / (VEC / 2) * (VEC / 2), heads = a.Hq + a.Hk, per_head = a.D / VEC;
    const int sv = RP_THREADS % per_head, sh = RP_THREADS / per_head % heads, st = RP_THREADS / per_head / heads;
    int v = threadIdx.x % per_head, h = threadIdx.x / per_head % heads, t = threadIdx.x / per_head / heads;
    bool first = true;
    do {
        Vec<T, VEC> x[BATCH];
        T* dst[BATCH];
        int at[BATCH], pair[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            dst[b] = nullptr;
            if (t < nt) {
                const bool isq = h < a.Hq;
                const int hh = isq ? h : h - a.Hq;
                const int64_t row = t0 + t;
                const T* src = (isq ? static_cast<const T*>(a.q) + row * a.q_stride_t + hh * a.q_stride_h
                                    : static_cast<const T*>(a.k) + row * a.k_stride_t + hh * a.k_stride_h);
                T* out = (isq ? static_cast<T*>(a.q_out) + row * a.qo_stride_t + hh * a.qo_stride_h
                              : static_cast<T*>(a.k_out) + row * a.ko_stride_t + hh * a.ko_stride_h);
                pair[b] = v * (VEC / 2);
                at[b] = t * slots + pair[b];
                dst[b] = out + v * VEC;
                x[b] = load_vec<T, VEC>(src + v * VEC);
                v += sv;
                h += sh;
                t += st;
                if (v >= per_head) {
                    v -= per_head;
                    ++h;
                }
                if (h >= heads) {
                    h -= heads;
                    ++t;
                }
            }
        }
        if (first) {                                         // (while the first items are on their way)
            turn_table(a, tab, pairs, slots, t0, nt, cs);
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            if (dst[b] == nullptr) continue;
            if (pair[b] >= pairs) {
                store_vec(dst[b], x[b]);
                continue;
            }
            float u[VEC], y[VEC];
            x[b].get(u);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
                const float2 w = cs[at[b] + e];              // cos, sin
                const bool turns = pair[b] + e < pairs;
                y[2 * e] = turns ? u[2 * e] * w.x - u[2 * e + 1] * w.y : u[2 * e];
                y[2 * e + 1] = turns ? u[2 * e + 1] * w.x + u[2 * e] * w.y : u[2 * e + 1];
            }
            x[b].set(y);
            store_vec(dst[b], x[b]);
        }
    } while (t < nt);
}

// Pairs (j, j + P), or unaligned ones: an item is VEC pairs of one head of one token (or VEC of the elements
// behind the pairs).
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS, 4) rope_kernel(const dn8_rope_args a, const __grid_constant__ RopeTable tab,
                                                          int pairs, int tokens_per_block) {
    extern __shared__ __align__(16) float2 cs[];  // [tokens of the block][pairs]
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
    const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.T - t0));
    const int heads = a.Hq + a.Hk;
    const int pv = pairs / VEC, tail = (a.D - 2 * pairs) / VEC, per_head = pv + tail;
    // Item i = (token, head, v). A thread's items are RP_THREADS apart: the three indices advance by
    // constant steps with a carry, instead of two divisions per item.
    const int sv = RP_THREADS % per_head, sh = RP_THREADS / per_head % heads, st = RP_THREADS / per_head / heads;
    int v = threadIdx.x % per_head, h = threadIdx.x / per_head % heads, t = threadIdx.x / per_head / heads;
    bool first = true;
    do {
        Vec<T, VEC> x1[RP_BATCH], x2[RP_BATCH];              // (interleaved: 2 VEC consecutive elements)
        T* dst[RP_BATCH];
        const float2* c[RP_BATCH];
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            dst[b] = nullptr;
            if (t < nt) {
                const bool isq = h < a.Hq;
                const int hh = isq ? h : h - a.Hq;
                const int64_t row = t0 + t;
                const T* src = (isq ? static_cast<const T*>(a.q) + row * a.q_stride_t + hh * a.q_stride_h
                                    : static_cast<const T*>(a.k) + row * a.k_stride_t + hh * a.k_stride_h);
                T* out = (isq ? static_cast<T*>(a.q_out) + row * a.qo_stride_t + hh * a.qo_stride_h
                              : static_cast<T*>(a.k_out) + row * a.ko_stride_t + hh * a.ko_stride_h);
                // where the item's elements start, and those of its other half
                const int at = v >= pv ? 2 * pairs + (v - pv) * VEC : INTER ? 2 * v * VEC : v * VEC;
                c[b] = v >= pv ? nullptr : cs + t * pairs + v * VEC;
                dst[b] = out + at;
                x1[b] = load_vec<T, VEC>(src + at);
                if (v < pv) x2[b] = load_vec<T, VEC>(src + at + (INTER ? VEC : pairs));
                v += sv;
                h += sh;
                t += st;
                if (v >= per_head) {
                    v -= per_head;
                    ++h;
                }
                if (h >= heads) {
                    h -= heads;
                    ++t;
                }
            }
        }
        if (first) {                                         // (while the first items are on their way)
            turn_table(a, tab, pairs, pairs, t0, nt, cs);
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            if (dst[b] == nullptr) continue;
            if (c[b] == nullptr) {
                store_vec(dst[b], x1[b]);
                continue;
            }
            float u[2 * VEC], y[2 * VEC];                    // the loaded elements in order, and the turned ones
            float (&lo)[VEC] = reinterpret_cast<float (&)[VEC]>(u);
            float (&hi)[VEC] = reinterpret_cast<float (&)[VEC]>(u[VEC]);
            x1[b].get(lo);
            x2[b].get(hi);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i1 = INTER ? 2 * e : e, i2 = INTER ? 2 * e + 1 : VEC + e;
                const float2 w = c[b][e];                    // cos, sin
                y[i1] = u[i1] * w.x - u[i2] * w.y;
                y[i2] = u[i2] * w.x + u[i1] * w.y;
            }
            x1[b].set(reinterpret_cast<const float (&)[VEC]>(y));
            x2[b].set(reinterpret_cast<const float (&)[VEC]>(y[VEC]));
            store_vec(dst[b], x1[b]);
            store_vec(dst[b] + (INTER ? VEC : pairs), x2[b]);
        }
    } while (t < nt);
}

// f_j / (2 pi) = base^(-e_j) / (2 pi): powers of one root per ladder, from two short tables of products
// (at most 8 + 16 roundings of 64 bits, instead of a pow() per pair).
static void ladder(double base, int n, int count, double* out) {
    const double root = std::pow(base, -1.0 / n);
    double lo[8], hi = 1.0;
    lo[0] = 0.15915494309189533577;               // 1 / (2 pi)
    for (int k = 1; k < 8; ++k) lo[k] = lo[k - 1] * root;
    const double r2 = root * root, r4 = r2 * r2, r8 = r4 * r4;
    for (int i = 0; i < count; ++i) {
        if (i && i % 8 == 0) hi *= r8;
        out[i] = lo[i % 8] * hi;
    }
}

cudaError_t launch_rope(const dn8_rope_args& a, int sms, cudaStream_t st) {
    RopeTable tab = {};
    int pairs = 0;
    for (int x = 0; x < a.n_axes; ++x) {
        for (int i = 0; i < a.sections[x]; ++i) tab.axis[pairs + i] = static_cast<uint8_t>(x);
        if (a.per_axis && a.sections[x] > 0) ladder(a.base, a.sections[x], a.sections[x], tab.turns + pairs);
        pairs += a.sections[x];
    }
    if (!a.per_axis) ladder(a.base, pairs, pairs, tab.turns);
    const int size = a.type == DN8_F32 ? 4 : 2, vec = 16 / size;
    const int heads = a.Hq + a.Hk;
    // 16-byte access where every head's pairs start on such a boundary, single elements otherwise
    const int64_t strides[] = {a.q_stride_t, a.q_stride_h, a.qo_stride_t, a.qo_stride_h,
                               a.k_stride_t, a.k_stride_h, a.ko_stride_t, a.ko_stride_h};
    bool wide = a.interleaved ? a.D % vec == 0 : pairs % vec == 0 && (a.D - 2 * pairs) % vec == 0;
    for (int k = 0; k < (a.Hk ? 8 : 4); ++k) wide = wide && strides[k] % vec == 0;
    for (const void* p : {a.q, static_cast<const void*>(a.q_out), a.k, static_cast<const void*>(a.k_out)})
        wide = wide && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    const int v = wide ? vec : 1;
    // Tokens per block: so many items per thread, but at least two blocks per SM while there
    // are tokens for them.
    const bool inter = wide && a.interleaved;
    const int per_token = heads * ((a.D + 2 * vec - 1) / (2 * vec));      // (of 16 bytes, single elements or not)
    const int slots = inter ? (pairs + v / 2 - 1) / (v / 2) * (v / 2) : pairs;
    int64_t tpb = RP_THREADS * (wide ? RP_BLOCK_WIDE : RP_BLOCK_NARROW) / (per_token > 0 ? per_token : 1);
    const int64_t spread = a.T / (2 * sms);
    if (tpb > spread) tpb = spread;
    if (tpb < 1) tpb = 1;
    if (tpb > 4096 / slots) tpb = 4096 / slots;              // 32 KB of cos / sin
    const int64_t blocks = (a.T + tpb - 1) / tpb;
    const size_t smem = static_cast<size_t>(tpb) * slots * sizeof(float2);
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int W = 16 / sizeof(T);
        auto kernel = wide ? (a.interleaved ? rope_inter_kernel<T, W> : rope_kernel<T, W, false>)
                           : (a.interleaved ? rope_kernel<T, 1, true> : rope_kernel<T, 1, false>);
        return launch_pdl(false, kernel, dim3(static_cast<unsigned>(blocks)), dim3(RP_THREADS), smem, st, a, tab, pairs,
                          static_cast<int>(tpb));
    });
}

}  // namespace dn8
