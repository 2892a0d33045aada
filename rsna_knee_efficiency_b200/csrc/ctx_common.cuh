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

// N consecutive elements as one unit of memory access (up to 16 bytes per instruction; the caller
// vouches for the alignment of N elements, or of 16 bytes where they are longer).
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };

template <typename T, int N> DN8_DEV void load_f32(const T* p, float (&f)[N]) {
    const Vec<T, N> t = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = to_f32(t.v[k]);
}
template <typename T, int N> DN8_DEV void store_f32(T* p, const float (&f)[N]) {
    Vec<T, N> t;
#pragma unroll
    for (int k = 0; k < N; ++k) t.v[k] = from_f32<T>(f[k]);
    *reinterpret_cast<Vec<T, N>*>(p) = t;
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
