// What the batched-decoding operators share: the two 16-bit types, eight values at a time.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ml2 {

template <typename T> struct Pair;
template <> struct Pair<__half> {
    using type = __half2;
    static __device__ __forceinline__ float2 up(__half2 v) { return __half22float2(v); }
    static __device__ __forceinline__ __half2 down(float a, float b) { return __floats2half2_rn(a, b); }
};
template <> struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ float2 up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
    static __device__ __forceinline__ __nv_bfloat162 down(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w)
{
    typename Pair<T>::type v;
    memcpy(&v, &w, 4);
    return Pair<T>::up(v);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const typename Pair<T>::type v = Pair<T>::down(a, b);
    uint32_t w;
    memcpy(&w, &v, 4);
    return w;
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8])
{
    const float2 a = unpack2<T>(v.x), b = unpack2<T>(v.y), c = unpack2<T>(v.z), d = unpack2<T>(v.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8])
{
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

}  // namespace ml2
