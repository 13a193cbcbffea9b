// Device side of the block-scaled FP8 format, shared by the quantiser and by the product that
// quantises its few rows itself: values in registers, block maxima, scales and codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace aeisu {
namespace blockq {

// Sixteen values of a row as they come: pairs of 16-bit values, or floats.
template <typename T> struct Vals {
    static constexpr int n = 8;               // values in 16 bytes
    uint32_t w[8];
    __device__ __forceinline__ float get(int i) const;
};
template <> struct Vals<float> {
    static constexpr int n = 4;
    float w[16];
    __device__ __forceinline__ float get(int i) const { return w[i]; }
};
template <> __device__ __forceinline__ float Vals<__nv_bfloat16>::get(int i) const {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}
template <> __device__ __forceinline__ float Vals<__half>::get(int i) const {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
    return i & 1 ? __high2float(h) : __low2float(h);
}

// Largest magnitudes, lane by lane of a pair; NaN does not count.  The pair of a float is itself alone.
template <typename T> struct Pair { using type = uint32_t; };
template <> struct Pair<float> { using type = float; };
template <typename T> __device__ __forceinline__ typename Pair<T>::type larger(typename Pair<T>::type a, typename Pair<T>::type b);
template <> __device__ __forceinline__ float larger<float>(float a, float b) { return fmaxf(fabsf(a), fabsf(b)); }
template <> __device__ __forceinline__ uint32_t larger<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)),
                                     __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <> __device__ __forceinline__ uint32_t larger<__half>(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(__habs2(*reinterpret_cast<const __half2*>(&a)), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
}
// The one or two values of a pair of maxima (NaN only where every value was: then zero).
__device__ __forceinline__ float number_or_zero(float v) { return fmaxf(v, 0.f); }
template <typename T> __device__ __forceinline__ float first_of(typename Pair<T>::type p);
template <typename T> __device__ __forceinline__ float second_of(typename Pair<T>::type p);
template <> __device__ __forceinline__ float first_of<float>(float p) { return number_or_zero(p); }
template <> __device__ __forceinline__ float second_of<float>(float) { return 0.f; }
template <> __device__ __forceinline__ float first_of<__nv_bfloat16>(uint32_t p) { return number_or_zero(__uint_as_float(p << 16)); }
template <> __device__ __forceinline__ float second_of<__nv_bfloat16>(uint32_t p) { return number_or_zero(__uint_as_float(p & 0xffff0000u)); }
template <> __device__ __forceinline__ float first_of<__half>(uint32_t p) { return number_or_zero(__low2float(*reinterpret_cast<const __half2*>(&p))); }
template <> __device__ __forceinline__ float second_of<__half>(uint32_t p) { return number_or_zero(__high2float(*reinterpret_cast<const __half2*>(&p))); }

// Eight consecutive values of a row, to places 8 h .. of v; columns at or past `cols` read as zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(Vals<T>& v, int h, const T* row, int c, int cols) {
    constexpr int n = Vals<T>::n;
    uint4* dst = reinterpret_cast<uint4*>(v.w) + h * (8 / n);
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 8 / n; ++i) {
            dst[i] = make_uint4(0, 0, 0, 0);
            if (c + i * n < cols) dst[i] = __ldg(reinterpret_cast<const uint4*>(row + c + i * n));
        }
    } else {
        T* e = reinterpret_cast<T*>(dst);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = c + i < cols ? row[c + i] : T(0.f);
    }
}

// Infinities to NaN, which the maxima ignore and the conversion keeps.
template <typename T>
__device__ __forceinline__ void infinities_to_nan(Vals<T>& v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (isinf(v.w[i])) v.w[i] = __uint_as_float(0x7fffffffu);
    } else {
        constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if ((v.w[i] & 0x7fffu) == inf) v.w[i] |= 0x7fffu;
            if ((v.w[i] >> 16 & 0x7fffu) == inf) v.w[i] |= 0x7fff0000u;
        }
    }
}

// Largest magnitude of the sixteen values, after infinities became NaN (a rare second pass).
template <typename T>
__device__ __forceinline__ float finite_max(Vals<T>& v) {
    auto largest = [&] {
        auto m = v.w[0];
#pragma unroll
        for (int i = 1; i < int(sizeof(v.w) / 4); ++i) m = larger<T>(m, v.w[i]);
        if constexpr (sizeof(T) == 4) return fmaxf(fabsf(m), 0.f);
        else return fmaxf(first_of<T>(m), second_of<T>(m));
    };
    float m = largest();
    if (isinf(m)) {
        infinities_to_nan(v);
        m = largest();
    }
    return m;
}

// The same of the first eight values and of the last eight.
template <typename T>
__device__ __forceinline__ void finite_max2(Vals<T>& v, float& first, float& second) {
    constexpr int n = sizeof(v.w) / 8;
    auto largest = [&](int from) {
        auto m = v.w[from];
#pragma unroll
        for (int i = 1; i < n; ++i) m = larger<T>(m, v.w[from + i]);
        if constexpr (sizeof(T) == 4) return fmaxf(fabsf(m), 0.f);
        else return fmaxf(first_of<T>(m), second_of<T>(m));
    };
    first = largest(0), second = largest(n);
    if (isinf(first) || isinf(second)) {
        infinities_to_nan(v);
        first = largest(0), second = largest(n);
    }
}

// Biased exponent of the scale.  amax = m 2^e with 0.5 <= m < 1 has the exponent field e + 126; the
// largest code is 0.875 * 2^top, so s = 2^(e - top), doubled where m > 0.875.
template <bool E5M2>
__device__ __forceinline__ uint32_t scale_of(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = int(b >> 23) + 1 - (E5M2 ? 16 : 9) + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b == 0 ? 127u : uint32_t(max(e, 0));
}
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    if constexpr (E5M2) {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    } else {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    }
    return uint32_t(lo) | (uint32_t(hi) << 16);
}

}  // namespace blockq
}  // namespace aeisu
