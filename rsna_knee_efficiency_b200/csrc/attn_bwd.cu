// attn_bwd.cu -- the gradient of attention (attn.cu): with P = exp(scale q k - lse) on the visible pairs
// and delta = sum(dout out) per row and head,
//   dv = P^T dout,  dS = P (dout v^T - delta) scale,  dq = dS k,  dk = dS^T q,
// dk and dv summed over the query heads of a key head's group. A query that sees nothing has lse =
// -inf: its P is taken as zero. No atomics: a row of dq is summed by one CTA over the keys, a row of
// dk, dv by one CTA over the queries, so the same inputs give the same bits.
#include "attn_common.cuh"

namespace dn8 {

template <typename T> __global__ void __launch_bounds__(256) attn_delta_kernel(const dn8_attention_bwd_args a) {
    const int64_t k = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (k >= a.Tq * a.Hq) return;
    const int64_t row = k / a.Hq, h = k % a.Hq;
    const T* o = static_cast<const T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h;
    const T* g = static_cast<const T*>(a.dout) + row * a.do_stride_t + h * a.do_stride_h;
    float s = 0.0f;
    for (int d = threadIdx.x & 31; d < a.D; d += 32) s = fmaf(to_f32(o[d]), to_f32(g[d]), s);
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) static_cast<float*>(a.work)[k] = s;
}

// One warp per query row and head; the lanes hold D / 32 elements each.
template <typename T> __global__ void __launch_bounds__(32) attn_dq_kernel(const dn8_attention_bwd_args a) {
    const int lane = threadIdx.x, h = blockIdx.y, kvh = h / (a.Hq / a.Hk);
    const Sequence sq = find_block<false>(a, blockIdx.x, 1, 1);
    if (sq.b < 0) return;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const int64_t row = sq.q0 + sq.blk;
    const int p = sq.blk + sq.nk - sq.nq;
    const float lse = a.lse[row * a.Hq + h], delta = static_cast<const float*>(a.work)[row * a.Hq + h];
    float q[4], g[4], acc[4] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 32 * e;
        q[e] = d < a.D ? to_f32((static_cast<const T*>(a.q) + row * a.q_stride_t + h * a.q_stride_h)[d]) : 0.0f;
        g[e] = d < a.D ? to_f32((static_cast<const T*>(a.dout) + row * a.do_stride_t + h * a.do_stride_h)[d]) : 0.0f;
    }
    const KeyTiles kt = key_tiles(p, p, sq.nk, left, right, a.sinks, 1);
    if (lse != -INFINITY)
        for (int t = 0; t < kt.count; ++t) {
            const int64_t j = kt.tile(t), at = sq.k0 + j;
            if (a.keep != nullptr && a.keep[at] == 0) continue;
            float k[4], s = 0.0f, dp = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = lane + 32 * e;
                k[e] = d < a.D ? to_f32((static_cast<const T*>(a.k) + at * a.k_stride_t + kvh * a.k_stride_h)[d]) : 0.0f;
                const float v = d < a.D ? to_f32((static_cast<const T*>(a.v) + at * a.v_stride_t + kvh * a.v_stride_h)[d]) : 0.0f;
                s = fmaf(q[e], k[e], s);
                dp = fmaf(g[e], v, dp);
            }
            const float ds = __expf(warp_sum(s) * a.scale - lse) * (warp_sum(dp) - delta) * a.scale;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(ds, k[e], acc[e]);
        }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.D)
            (static_cast<T*>(a.dq) + row * a.dq_stride_t + h * a.dq_stride_h)[lane + 32 * e] = from_f32<T>(acc[e]);
}

// One warp per key row and key head.
template <typename T> __global__ void __launch_bounds__(32) attn_dkv_kernel(const dn8_attention_bwd_args a) {
    const int lane = threadIdx.x, kvh = blockIdx.y, G = a.Hq / a.Hk;
    const Sequence sq = find_block<true>(a, blockIdx.x, 1, 1);
    if (sq.b < 0) return;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const int j = sq.blk, off = sq.nk - sq.nq;
    const int64_t at = static_cast<int64_t>(sq.k0) + j;
    float k[4], v[4], dk[4] = {}, dv[4] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 32 * e;
        k[e] = d < a.D ? to_f32((static_cast<const T*>(a.k) + at * a.k_stride_t + kvh * a.k_stride_h)[d]) : 0.0f;
        v[e] = d < a.D ? to_f32((static_cast<const T*>(a.v) + at * a.v_stride_t + kvh * a.v_stride_h)[d]) : 0.0f;
    }
    if (a.keep == nullptr || a.keep[at] != 0)
        for (int i = max(0, j - right - off); i < sq.nq; ++i) {
            const int p = i + off;
            if (j < p - left && j >= a.sinks) break;
            const int64_t row = sq.q0 + i;
            for (int h = kvh * G; h < kvh * G + G; ++h) {
                const float lse = a.lse[row * a.Hq + h];
                if (lse == -INFINITY) continue;
                float q[4], g[4], s = 0.0f, dp = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = lane + 32 * e;
                    q[e] = d < a.D ? to_f32((static_cast<const T*>(a.q) + row * a.q_stride_t + h * a.q_stride_h)[d]) : 0.0f;
                    g[e] = d < a.D ? to_f32((static_cast<const T*>(a.dout) + row * a.do_stride_t + h * a.do_stride_h)[d]) : 0.0f;
                    s = fmaf(q[e], k[e], s);
                    dp = fmaf(g[e], v[e], dp);
                }
                const float pr = __expf(warp_sum(s) * a.scale - lse);
                const float ds = pr * (warp_sum(dp) - static_cast<const float*>(a.work)[row * a.Hq + h]) * a.scale;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dk[e] = fmaf(ds, q[e], dk[e]);
                    dv[e] = fmaf(pr, g[e], dv[e]);
                }
            }
        }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.D) {
            (static_cast<T*>(a.dk) + at * a.dk_stride_t + kvh * a.dk_stride_h)[lane + 32 * e] = from_f32<T>(dk[e]);
            (static_cast<T*>(a.dv) + at * a.dv_stride_t + kvh * a.dv_stride_h)[lane + 32 * e] = from_f32<T>(dv[e]);
        }
}

size_t attention_bwd_work(const dn8_attention_bwd_args& a) { return static_cast<size_t>(a.Tq) * a.Hq * sizeof(float); }

template <typename T> static cudaError_t bwd_go(const dn8_attention_bwd_args& a, cudaStream_t st) {
    if (a.Tq > 0) {
        cudaError_t e = launch_pdl(false, attn_delta_kernel<T>, dim3(static_cast<unsigned>((a.Tq * a.Hq + 7) / 8)), dim3(256),
                                   0, st, a);
        if (e != cudaSuccess) return e;
        e = launch_pdl(false, attn_dq_kernel<T>, dim3(static_cast<unsigned>(a.Tq), a.Hq), dim3(32), 0, st, a);
        if (e != cudaSuccess) return e;
    }
    if (a.Tk == 0) return cudaSuccess;
    return launch_pdl(false, attn_dkv_kernel<T>, dim3(static_cast<unsigned>(a.Tk), a.Hk), dim3(32), 0, st, a);
}

cudaError_t launch_attention_bwd(const dn8_attention_bwd_args& a, int sms, cudaStream_t st) {
    (void)sms;
    return a.type == DN8_F16 ? bwd_go<__half>(a, st) : bwd_go<__nv_bfloat16>(a, st);
}

}  // namespace dn8
