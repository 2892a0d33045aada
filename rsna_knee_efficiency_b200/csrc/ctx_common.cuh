// ctx_common.cuh -- element types and vector access shared by the context transformer's kernels
// (layer norm, rotary positions, attention).
#pragma once
#include <cuda_bf16.h>

#include "../../include/dn8.h"
#include "dn8_common.cuh"

namespace dn8 {

DN8_DEV float to_f32(float v) { return v; }
DN8_DEV float to_f32(__half v) { return __half2float(v); }
DN8_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> DN8_DEV T from_f32(float v);
template <> DN8_DEV float from_f32<float>(float v) { return v; }
template <> DN8_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> DN8_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

DN8_DEV uint32_t pack2(__half, float lo, float hi) { return u32_of(__floats2half2_rn(lo, hi)); }
DN8_DEV uint32_t pack2(__nv_bfloat16, float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
DN8_DEV float2 unpack2(__half, uint32_t u) { return __half22float2(h2_of(u)); }
DN8_DEV float2 unpack2(__nv_bfloat16, uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

// N consecutive elements as one unit of memory access (up to 16 bytes per instruction; the caller
// vouches for the alignment of N elements, or of 16 bytes where they are longer). Held as 32-bit words:
// as an array of 16-bit elements the compiler takes a register for each.
template <typename T, int N, bool WORDS = (sizeof(T) * N >= 4)>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
    uint32_t w[sizeof(T) * N / 4];
    DN8_DEV void get(float (&f)[N]) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (sizeof(T) == 4) {
                f[k] = __uint_as_float(w[k]);
            } else if (k % 2 == 0) {
                const float2 p = unpack2(T(), w[k / 2]);
                f[k] = p.x;
                f[k + 1] = p.y;
            }
        }
    }
    DN8_DEV void set(const float (&f)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(f[k]);
            else if (k % 2 == 0) w[k / 2] = pack2(T(), f[k], f[k + 1]);
        }
    }
};
template <typename T, int N> struct Vec<T, N, false> {
    T v;
    DN8_DEV void get(float (&f)[N]) const { f[0] = to_f32(v); }
    DN8_DEV void set(const float (&f)[N]) { v = from_f32<T>(f[0]); }
};
template <typename T, int N> DN8_DEV Vec<T, N> load_vec(const T* p) { return *reinterpret_cast<const Vec<T, N>*>(p); }
template <typename T, int N> DN8_DEV void store_vec(T* p, const Vec<T, N>& v) { *reinterpret_cast<Vec<T, N>*>(p) = v; }

template <typename T, int N> DN8_DEV void load_f32(const T* p, float (&f)[N]) { load_vec<T, N>(p).get(f); }
template <typename T, int N> DN8_DEV void store_f32(T* p, const float (&f)[N]) {
    Vec<T, N> t;
    t.set(f);
    store_vec(p, t);
}
// N weights (or biases) of type DN8_F32 / DN8_F16 / DN8_BF16 at element `at` (N > 1: 16-byte aligned)
template <int N> DN8_DEV void load_param(const void* p, int type, int at, float (&f)[N]) {
    if (type == DN8_F32) load_f32(static_cast<const float*>(p) + at, f);
    else if (type == DN8_F16) load_f32(static_cast<const __half*>(p) + at, f);
    else load_f32(static_cast<const __nv_bfloat16*>(p) + at, f);
}

DN8_DEV float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Calls f.template operator()<T>() for the element type `type`.
template <typename F> cudaError_t with_type(int type, F&& f) {
    switch (type) {
        case DN8_F32: return f(float());
        case DN8_F16: return f(__half());
        default: return f(__nv_bfloat16());
    }
}

}  // namespace dn8
