// Eight consecutive elements of a row of bf16, float16 or float32, in float32 registers.
#pragma once
#include "mi8_half.h"

namespace mi8 {

template <typename T>
struct Eight {  // bf16, float16
    static constexpr int kBytes = 2;
    uint4 v;
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = T::lo(w[e]);
            f[2 * e + 1] = T::hi(w[e]);
        }
    }
    // elements c .. c + 7 of a row of n, zeros past it; WIDE: whole 16-byte chunks
    template <bool WIDE>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        v = make_uint4(0, 0, 0, 0);
        const uint16_t* p = static_cast<const uint16_t*>(row) + c;
        if constexpr (WIDE) {
            if (c < n) v = *reinterpret_cast<const uint4*>(p);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = c + e < n ? p[e] : 0;
            v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
    }
    template <bool WIDE>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        uint16_t* p = static_cast<uint16_t*>(row) + c;
        const uint32_t w[4] = {T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7])};
        if constexpr (WIDE) {
            if (c < n) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < n) p[e] = (uint16_t)(w[e >> 1] >> 16 * (e & 1));
        }
    }
};

struct F32 {
    static constexpr int kCode = MI8_F32;
};
template <>
struct Eight<F32> {
    static constexpr int kBytes = 4;
    float4 a, b;
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    template <bool WIDE>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        a = b = make_float4(0, 0, 0, 0);
        const float* p = static_cast<const float*>(row) + c;
        if constexpr (WIDE) {
            if (c < n) {
                a = *reinterpret_cast<const float4*>(p);
                b = *reinterpret_cast<const float4*>(p + 4);
            }
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = c + e < n ? p[e] : 0.0f;
            a = make_float4(f[0], f[1], f[2], f[3]);
            b = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
    template <bool WIDE>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        float* p = static_cast<float*>(row) + c;
        if constexpr (WIDE) {
            if (c < n) {
                *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < n) p[e] = f[e];
        }
    }
};

inline int bytes_of(int hp_dtype) { return hp_dtype == MI8_F32 ? 4 : 2; }
inline bool float_type(int hp_dtype) { return hp_dtype == MI8_BF16 || hp_dtype == MI8_F16 || hp_dtype == MI8_F32; }

}  // namespace mi8
