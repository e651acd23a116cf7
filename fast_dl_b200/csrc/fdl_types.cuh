// Element types of the operators that take 32-bit or 16-bit tensors: 128-bit packs of either,
// unpacked to and rounded from 32-bit registers (all arithmetic is in 32 bits or more; the one
// rounding to 16 bits is the store of a result, to nearest even).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fdl_common.cuh"

namespace fdl {

inline bool known_dtype(int dtype) { return dtype == FDL_F32 || dtype == FDL_F16 || dtype == FDL_BF16; }
inline size_t dtype_bytes(int dtype) { return dtype == FDL_F32 ? 4 : 2; }

#ifdef __CUDACC__

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T>
constexpr int kPack = 16 / static_cast<int>(sizeof(T));  // elements of a 128-bit pack

__device__ __forceinline__ void unpack(const uint4& u, float (&v)[4], float) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __half) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __nv_bfloat16) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bfloat16 is the upper half of the float of the same value
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ uint4 repack(const float (&v)[4], float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 repack(const float (&v)[8], __half) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 repack(const float (&v)[8], __nv_bfloat16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// N consecutive elements as floats: one 128-bit access (N == kPack<T>, aligned) or one element (N == 1).
template <class T, int N>
struct Chunk {
    static_assert(N == kPack<T>, "a chunk is one 128-bit pack, or one element");
    __device__ static __forceinline__ void load(const T* p, float (&v)[N]) {
        unpack(*reinterpret_cast<const uint4*>(p), v, T{});
    }
    __device__ static __forceinline__ void load_stream(const T* p, float (&v)[N]) {
        unpack(__ldcs(reinterpret_cast<const uint4*>(p)), v, T{});
    }
    __device__ static __forceinline__ void store_stream(T* p, const float (&v)[N]) {
        __stcs(reinterpret_cast<uint4*>(p), repack(v, T{}));
    }
};
template <class T>
struct Chunk<T, 1> {
    __device__ static __forceinline__ void load(const T* p, float (&v)[1]) { v[0] = to_f32(*p); }
    __device__ static __forceinline__ void load_stream(const T* p, float (&v)[1]) { v[0] = to_f32(__ldcs(p)); }
    __device__ static __forceinline__ void store_stream(T* p, const float (&v)[1]) { __stcs(p, from_f32<T>(v[0])); }
};

// Two floats in one instruction (a rounding each, as for one).
__device__ __forceinline__ uint64_t bits2(float2 v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 floats2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
    return floats2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
    return floats2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
    return floats2(d);
}

// A 128-bit pack as pairs.
__device__ __forceinline__ void unpack2(const uint4& u, float2 (&v)[2], float) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ void unpack2(const uint4& u, float2 (&v)[4], __half) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
__device__ __forceinline__ void unpack2(const uint4& u, float2 (&v)[4], __nv_bfloat16) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <class T, int M>
__device__ __forceinline__ void store_pairs(T* p, const float2 (&v)[M]) {
    float f[2 * M];
#pragma unroll
    for (int e = 0; e < M; ++e) {
        f[2 * e] = v[e].x;
        f[2 * e + 1] = v[e].y;
    }
    __stcs(reinterpret_cast<uint4*>(p), repack(f, T{}));
}
// 2^x with a relative error of about 2^-22.
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

#endif  // __CUDACC__

// Calls fn with a null pointer of the element type that `dtype` names (known_dtype holds).
template <class Fn>
int with_dtype(int dtype, Fn&& fn) {
    if (dtype == FDL_F32) return fn(static_cast<float*>(nullptr));
    if (dtype == FDL_F16) return fn(static_cast<__half*>(nullptr));
    return fn(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace fdl
