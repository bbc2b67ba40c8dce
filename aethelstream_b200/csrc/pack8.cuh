// pack8.cuh -- eight features of a row in registers, in the type that they have
// in memory.
#pragma once
#include "common.cuh"

namespace aeth {

// Eight consecutive features of a row as they lie in memory.
template <typename T>
struct Pack8 {
    static constexpr int kWords = (int)sizeof(T) / 2;
    uint4 w[kWords];
};

template <typename T>
__device__ __forceinline__ float ck_value(const Pack8<T>& p, int i);
template <>
__device__ __forceinline__ float ck_value<float>(const Pack8<float>& p, int i) {
    const uint4 q = p.w[i >> 2];
    return __uint_as_float((i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w);
}
template <>
__device__ __forceinline__ float ck_value<__nv_bfloat16>(const Pack8<__nv_bfloat16>& p, int i) {
    const uint4 q = p.w[0];
    const uint32_t x = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __uint_as_float((i & 1) ? x & 0xffff0000u : x << 16);
}
template <>
__device__ __forceinline__ float ck_value<__half>(const Pack8<__half>& p, int i) {
    const uint4 q = p.w[0];
    const uint32_t x = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __half2float(__ushort_as_half((uint16_t)((i & 1) ? x >> 16 : x)));
}

template <typename T>
__device__ __forceinline__ uint32_t ck_pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t ck_pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t ck_pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ Pack8<T> ck_pack(const float (&v)[8]) {
    Pack8<T> p;
    if constexpr (sizeof(T) == 4) {
        p.w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        p.w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        p.w[0] = make_uint4(ck_pack2<T>(v[0], v[1]), ck_pack2<T>(v[2], v[3]), ck_pack2<T>(v[4], v[5]),
                            ck_pack2<T>(v[6], v[7]));
    }
    return p;
}

// Read once: past L1, so that it keeps the gain.
__device__ __forceinline__ uint4 ck_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ck_stream(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// -r^3 mean(dy gain x), what x is taken times in a norm's dx.  r |mean| is at most the root
// mean square of dy gain, so that one factor of r at a time stays in fp32's range as long
// as r^2 does (r^3 leaves it where activations reach 1e13, or 1e-13 without eps).
__device__ __forceinline__ float ck_back_factor(float r, float mean) { return -(r * (r * (r * mean))); }

}  // namespace aeth
