// Rows stored as fp32, bf16 or fp16 and computed in fp32: vector loads and stores, warp and block sums in a fixed order.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace e3b {

enum DataType { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };   // codes of the C entry points

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 load(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
    static __device__ __forceinline__ uint32_t store(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 load(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    static __device__ __forceinline__ uint32_t store(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};

template <typename T> __device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <typename T> __device__ __forceinline__ T from_float(float v) { return T(v); }

// VEC consecutive elements as they lie in memory (one load), and their fp32 values.
template <typename T, int VEC> struct Packed;
template <typename T> struct Packed<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void zero() { v = from_float<T>(0.0f); }
    __device__ __forceinline__ void unpack(float* f) const { f[0] = to_float(v); }
    static __device__ __forceinline__ void store(T* p, const float* f) { *p = from_float<T>(f[0]); }
};
template <> struct Packed<float, 2> {
    float2 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float2*>(p); }
    __device__ __forceinline__ void unpack(float* f) const { f[0] = v.x; f[1] = v.y; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]); }
};
template <typename T> struct Packed<T, 2> {
    uint32_t v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint32_t*>(p); }
    __device__ __forceinline__ void unpack(float* f) const {
        const float2 a = Pair<T>::load(v);
        f[0] = a.x; f[1] = a.y;
    }
    static __device__ __forceinline__ void store(T* p, const float* f) { *reinterpret_cast<uint32_t*>(p) = Pair<T>::store(f[0], f[1]); }
};
template <> struct Packed<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void zero() { v = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void unpack(float* f) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <typename T> struct Packed<T, 4> {
    uint2 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void zero() { v = make_uint2(0u, 0u); }
    __device__ __forceinline__ void unpack(float* f) const {
        const float2 a = Pair<T>::load(v.x), b = Pair<T>::load(v.y);
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
    static __device__ __forceinline__ void store(T* p, const float* f) {
        *reinterpret_cast<uint2*>(p) = make_uint2(Pair<T>::store(f[0], f[1]), Pair<T>::store(f[2], f[3]));
    }
};

template <typename T> struct Packed<T, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void unpack(float* f) const {
        const float2 a = Pair<T>::load(v.x), b = Pair<T>::load(v.y), c = Pair<T>::load(v.z), d = Pair<T>::load(v.w);
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
    }
    static __device__ __forceinline__ void store(T* p, const float* f) {
        *reinterpret_cast<uint4*>(p) = make_uint4(Pair<T>::store(f[0], f[1]), Pair<T>::store(f[2], f[3]), Pair<T>::store(f[4], f[5]),
                                                  Pair<T>::store(f[6], f[7]));
    }
};
template <> struct Packed<float, 8> {
    float4 lo, hi;
    __device__ __forceinline__ void load(const float* p) {
        lo = *reinterpret_cast<const float4*>(p);
        hi = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void zero() { lo = hi = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void unpack(float* f) const {
        f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w; f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
    }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
};

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
// d = a * b + c and d = a * b over N columns (N even: by pairs)
template <int N>
__device__ __forceinline__ void fma_n(const float (&a)[N], const float (&b)[N], const float (&c)[N], float (&d)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
            d[i] = r.x;
            d[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = fmaf(a[i], b[i], c[i]);
    }
}
template <int N>
__device__ __forceinline__ void mul_n(const float (&a)[N], const float (&b)[N], float (&d)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 r = mul2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
            d[i] = r.x;
            d[i + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = a[i] * b[i];
    }
}
template <int N>
__device__ __forceinline__ void scale_n(const float (&a)[N], float by, float (&d)[N]) {
    float b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = by;
    mul_n<N>(a, b, d);
}
// sum of a * b
template <int N>
__device__ __forceinline__ float dot_n(const float (&a)[N], const float (&b)[N]) {
    if constexpr (N % 2 == 0) {
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < N; i += 2) s = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
        return s.x + s.y;
    } else {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
        return s;
    }
}
template <int N>
__device__ __forceinline__ void load_n(const float* p, float (&f)[N]) {
    Packed<float, N> v;
    v.load(p);
    v.unpack(f);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int N> using Int = std::integral_constant<int, N>;   // a size handed to a generic lambda

inline int element_size(int type) { return type == kFloat32 ? 4 : 2; }
inline bool known_type(int type) { return type >= kFloat32 && type <= kFloat16; }
// Whether vectors of `bytes` bytes may start at p.
inline bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace e3b
