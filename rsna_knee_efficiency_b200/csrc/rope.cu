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
// shared memory, computed once per (token, pair) and used by every head of q and k.
#include <cmath>

#include "ctx_common.cuh"
#include "dn8_kernels.h"

namespace dn8 {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_PAIRS = 128;
constexpr int RP_BATCH = 4;                       // items a thread has in flight

struct RopeTable {
    double turns[RP_MAX_PAIRS];                   // f_j / (2 pi)
    uint8_t axis[RP_MAX_PAIRS];
};

// An item is VEC pairs of one head of one token (or VEC of the elements behind the pairs).
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS) rope_kernel(const dn8_rope_args a, const __grid_constant__ RopeTable tab,
                                                          int pairs, int tokens_per_block) {
    extern __shared__ float2 cs[];                // [tokens of the block][pairs]
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
    const int nt = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), a.T - t0));
    for (int k = threadIdx.x; k < nt * pairs; k += RP_THREADS) {
        const int t = k / pairs, j = k - t * pairs;
        const double ang = static_cast<double>(a.pos[(t0 + t) * a.n_axes + tab.axis[j]]) * tab.turns[j];
        const float fr = static_cast<float>(2.0 * (ang - rint(ang)));      // half turns in [-1, 1]
        float s, c;
        sincospif(fr, &s, &c);
        cs[k] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    const int heads = a.Hq + a.Hk;
    const int pv = pairs / VEC, tail = (a.D - 2 * pairs) / VEC, per_head = pv + tail;
    const int items = nt * heads * per_head;
    for (int i0 = threadIdx.x; i0 < items; i0 += RP_THREADS * RP_BATCH) {
        float x1[RP_BATCH][VEC], x2[RP_BATCH][VEC];
        T* dst[RP_BATCH];
        int at[RP_BATCH], tok[RP_BATCH];
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            const int i = i0 + b * RP_THREADS;
            dst[b] = nullptr;
            if (i >= items) continue;
            const int v = i % per_head, th = i / per_head;
            const int h = th % heads;
            tok[b] = th / heads;
            const T* src;
            if (h < a.Hq) {
                src = static_cast<const T*>(a.q) + (t0 + tok[b]) * a.q_stride_t + h * a.q_stride_h;
                dst[b] = static_cast<T*>(a.q_out) + (t0 + tok[b]) * a.qo_stride_t + h * a.qo_stride_h;
            } else {
                src = static_cast<const T*>(a.k) + (t0 + tok[b]) * a.k_stride_t + (h - a.Hq) * a.k_stride_h;
                dst[b] = static_cast<T*>(a.k_out) + (t0 + tok[b]) * a.ko_stride_t + (h - a.Hq) * a.ko_stride_h;
            }
            if (v >= pv) {
                at[b] = -(2 * pairs + (v - pv) * VEC);
                load_f32(src - at[b], x1[b]);
            } else if (INTER) {
                at[b] = v * VEC;
                float x[2 * VEC];
                load_f32(src + 2 * at[b], x);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    x1[b][e] = x[2 * e];
                    x2[b][e] = x[2 * e + 1];
                }
            } else {
                at[b] = v * VEC;
                load_f32(src + at[b], x1[b]);
                load_f32(src + pairs + at[b], x2[b]);
            }
        }
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            if (dst[b] == nullptr) continue;
            if (at[b] < 0) {
                store_f32(dst[b] - at[b], x1[b]);
                continue;
            }
            const float2* c = cs + tok[b] * pairs + at[b];
            float y1[VEC], y2[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                y1[e] = x1[b][e] * c[e].x - x2[b][e] * c[e].y;
                y2[e] = x2[b][e] * c[e].x + x1[b][e] * c[e].y;
            }
            if (INTER) {
                float y[2 * VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    y[2 * e] = y1[e];
                    y[2 * e + 1] = y2[e];
                }
                store_f32(dst[b] + 2 * at[b], y);
            } else {
                store_f32(dst[b] + at[b], y1);
                store_f32(dst[b] + pairs + at[b], y2);
            }
        }
    }
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
    bool wide = pairs % vec == 0 && (a.D - 2 * pairs) % vec == 0;
    for (int k = 0; k < (a.Hk ? 8 : 4); ++k) wide = wide && strides[k] % vec == 0;
    for (const void* p : {a.q, static_cast<const void*>(a.q_out), a.k, static_cast<const void*>(a.k_out)})
        wide = wide && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    const int v = wide ? vec : 1;
    // Tokens per block: about RP_BATCH items per thread, but at least two blocks per SM while there
    // are tokens for them.
    const int per_token = heads * (pairs / v + (a.D - 2 * pairs) / v);
    int64_t tpb = RP_THREADS * RP_BATCH / (per_token > 0 ? per_token : 1);
    const int64_t spread = a.T / (2 * sms);
    if (tpb > spread) tpb = spread;
    if (tpb < 1) tpb = 1;
    if (tpb > 4096 / pairs) tpb = 4096 / pairs;              // 32 KB of cos / sin
    const int64_t blocks = (a.T + tpb - 1) / tpb;
    const size_t smem = static_cast<size_t>(tpb) * pairs * sizeof(float2);
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int W = 16 / sizeof(T);
        auto kernel = wide ? (a.interleaved ? rope_kernel<T, W, true> : rope_kernel<T, W, false>)
                           : (a.interleaved ? rope_kernel<T, 1, true> : rope_kernel<T, 1, false>);
        return launch_pdl(false, kernel, dim3(static_cast<unsigned>(blocks)), dim3(RP_THREADS), smem, st, a, tab, pairs,
                          static_cast<int>(tpb));
    });
}

}  // namespace dn8
