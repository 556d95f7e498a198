// Loads and stores of VEC consecutive channels of a 16-bit or float32 buffer as float32 values, in
// accesses of up to 16 bytes.
#pragma once

#include <cstdint>

#include "sm100.cuh"

namespace cflk {

inline bool aligned16(const void* p) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

template <>
struct Elem<float> {
    static __device__ __forceinline__ float to_f(float x) { return x; }
    static __device__ __forceinline__ float from_f(float x) { return x; }
};

// VEC channels as they are in memory, for loads that are kept in flight (8 or 16 bytes)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Raw {
    static constexpr int kWords = (int)sizeof(T) * VEC / 4;
    uint32_t w[kWords];
};

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T* p) {
    Raw<T, VEC> r;
    if constexpr (Raw<T, VEC>::kWords == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        r.w[0] = x.x;
        r.w[1] = x.y;
        r.w[2] = x.z;
        r.w[3] = x.w;
    } else {
        static_assert(Raw<T, VEC>::kWords == 2);
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        r.w[0] = x.x;
        r.w[1] = x.y;
    }
    return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack_raw(const Raw<T, VEC>& r, float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < Raw<T, VEC>::kWords; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(r.w[i]);
        } else {
            const float2 x = Elem<T>::unpack(r.w[i]);
            v[2 * i] = x.x;
            v[2 * i + 1] = x.y;
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = Elem<T>::to_f(p[0]);
    } else if constexpr (sizeof(T) == 4) {
        static_assert(VEC % 4 == 0);
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            const float4 w = reinterpret_cast<const float4*>(p)[i];
            v[4 * i] = w.x;
            v[4 * i + 1] = w.y;
            v[4 * i + 2] = w.z;
            v[4 * i + 3] = w.w;
        }
    } else if constexpr (VEC == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const float2 a = Elem<T>::unpack(w.x), b = Elem<T>::unpack(w.y);
        v[0] = a.x;
        v[1] = a.y;
        v[2] = b.x;
        v[3] = b.y;
    } else {
        static_assert(VEC == 8);
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = Elem<T>::unpack(q[i]);
            v[2 * i] = a.x;
            v[2 * i + 1] = a.y;
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = Elem<T>::from_f(v[0]);
    } else if constexpr (sizeof(T) == 4 && VEC == 8) {
        // one 32-byte access (p 32-byte aligned): two of 16 would each write half sectors
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]),
                     "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
    } else if constexpr (sizeof(T) == 4) {
        static_assert(VEC == 4);
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (VEC == 4) {
        *reinterpret_cast<uint2*>(p) =
            make_uint2(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]));
    } else {
        static_assert(VEC == 8);
        *reinterpret_cast<uint4*>(p) =
            make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]),
                       Elem<T>::pack(v[4], v[5]), Elem<T>::pack(v[6], v[7]));
    }
}

}  // namespace cflk
