// What the operators of a decoder's step share: refusals, vectors of 16 bytes as floats, the device's SM count.
// Whatever they are given (tables, scales, gains, weights) may be what the launch before writes: it is read behind pdl_enter(), by ordinary loads, since
// the non-coherent ones (__ldg) are for what stays as it is from a kernel's start on, and a kernel may be started under the launch before.
#pragma once
#include "common.cuh"

// a refusal with its reason, which goes where failed launches leave theirs
inline int thb_refuse(int code, const char *why)
{
    thb_note_launch(cudaErrorInvalidValue, why);
    return code;
}
inline bool thb_misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

inline int thb_sm_count()  // of the current device
{
    static int sms[64];
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && sms[dev]) return sms[dev];
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
    if (dev >= 0 && dev < 64) sms[dev] = n;
    return n;
}

// 16 bytes of a type as floats, and back with one rounding each
template <typename T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4 &t, float *v)
    {
        v[0] = __uint_as_float(t.x); v[1] = __uint_as_float(t.y); v[2] = __uint_as_float(t.z); v[3] = __uint_as_float(t.w);
    }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <typename T, typename T2> struct Vec16Half {
    static constexpr int N = 8;
    static __device__ __forceinline__ float2 wide(__half2 h) { return __half22float2(h); }
    static __device__ __forceinline__ float2 wide(__nv_bfloat162 h) { return __bfloat1622float2(h); }
    static __device__ __forceinline__ void narrow(float a, float b, __half2 *h) { *h = __floats2half2_rn(a, b); }
    static __device__ __forceinline__ void narrow(float a, float b, __nv_bfloat162 *h) { *h = __floats2bfloat162_rn(a, b); }
    static __device__ __forceinline__ void unpack(const uint4 &t, float *v)
    {
        const T2 *h = reinterpret_cast<const T2 *>(&t);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = wide(h[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        uint4 t;
        T2 *h = reinterpret_cast<T2 *>(&t);
#pragma unroll
        for (int i = 0; i < 4; i++) narrow(v[2 * i], v[2 * i + 1], h + i);
        return t;
    }
};
template <> struct Vec16<__half> : Vec16Half<__half, __half2> {};
template <> struct Vec16<__nv_bfloat16> : Vec16Half<__nv_bfloat16, __nv_bfloat162> {};

const char *thb_kv_cache_fault(const thb_kv_cache *c);  // kv_append.cu
