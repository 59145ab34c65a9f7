// What the kernels of the layer's dense operators share: element types, 16-byte loads and stores of them as fp32.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace lutamm {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);   // to nearest
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {   // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16*) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <typename T> constexpr int kPer16 = 16 / (int)sizeof(T);   // elements of 16 bytes

// E elements as fp32: 16 bytes at once (E = kPer16), or one.
template <typename T, int E>
__device__ __forceinline__ void load_elems(const T* p, float (&v)[E]) {
    if constexpr (E == 1) {
        v[0] = to_float(*p);
    } else {
        static_assert(E == kPer16<T>);
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
        } else {
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2(u[i], static_cast<T*>(nullptr));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[E]) {
    if constexpr (E == 1) {
        *p = from_float<T>(v[0]);
    } else {
        static_assert(E == kPer16<T>);
        uint4 w;
        if constexpr (sizeof(T) == 4) {
            w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        } else {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = pack2(v[2 * i], v[2 * i + 1], static_cast<T*>(nullptr));
            w = make_uint4(u[0], u[1], u[2], u[3]);
        }
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// E elements as they lie in memory.
template <typename T, int E>
struct Piece {
    uint4 w;
    __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void widen(float (&v)[E]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(u[i]);
            } else {
                const float2 f = unpack2(u[i], static_cast<T*>(nullptr));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};
template <typename T>
struct Piece<T, 1> {
    T w;
    __device__ __forceinline__ void load(const T* p) { w = *p; }
    __device__ __forceinline__ void widen(float (&v)[1]) const { v[0] = to_float(w); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace lutamm
