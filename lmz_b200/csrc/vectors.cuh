// Element types of a checkpoint's tensors, and vectors of them as memory instructions move them.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lmz {

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<1> { using type = uint8_t; };

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// Two in a word, the first in its lower half.
template <class T>
__device__ __forceinline__ uint32_t narrow_two(float lo, float hi)
{
    uint32_t word;
    if constexpr (__is_same(T, __half)) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(word) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(word) : "f"(hi), "f"(lo));
    return word;
}

// VB bytes of T as a memory instruction moves them.
template <class T, int VB>
struct Vec {
    static constexpr int N = VB / sizeof(T);
    union {
        typename Raw<VB>::type raw;
        T e[N];
    };
    __device__ __forceinline__ Vec() {}
};

// A vector's elements in 32 bits: of two BF16 in a word each is one instruction away.
template <class T, int VB>
__device__ __forceinline__ void widen_all(const Vec<T, VB> &v, float *to)
{
    if constexpr (__is_same(T, __nv_bfloat16) && VB >= 4) {
        union { typename Raw<VB>::type raw; uint32_t word[VB / 4]; } w;
        w.raw = v.raw;
#pragma unroll
        for (int e = 0; e < VB / 4; e++) to[2 * e] = __uint_as_float(w.word[e] << 16), to[2 * e + 1] = __uint_as_float(w.word[e] & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int e = 0; e < Vec<T, VB>::N; e++) to[e] = widen(v.e[e]);
    }
}

// And back, each rounded once: two to an instruction where there are two to a word.
template <class T, int VB>
__device__ __forceinline__ void narrow_all(const float *from, Vec<T, VB> &v)
{
    if constexpr (sizeof(T) == 2 && VB >= 4) {
        union { typename Raw<VB>::type raw; uint32_t word[VB / 4]; } w;
#pragma unroll
        for (int e = 0; e < VB / 4; e++) w.word[e] = narrow_two<T>(from[2 * e], from[2 * e + 1]);
        v.raw = w.raw;
    } else {
#pragma unroll
        for (int e = 0; e < Vec<T, VB>::N; e++) v.e[e] = narrow<T>(from[e]);
    }
}

}  // namespace lmz
