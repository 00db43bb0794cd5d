// Eight consecutive elements of a row of bf16, float16 or float32, in float32 registers.
//
// A lane's eight elements are one access of 16 bytes (two in float32) at any address: gfx950 serves global loads and stores at the alignment of the element, so
// rows of odd length need no other kernel, only their last chunk an element at a time (16-bit elements one by one instead: gradient of the epilogue,
// 1537 x 2771, 48 us).
#pragma once
#include "mi8_half.h"

namespace mi8 {

typedef uint32_t chunk16_t __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's alignment
typedef float chunk32_t __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
struct Eight {  // bf16, float16
    static constexpr int kBytes = 2;
    u32x4_t v;
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = T::lo(v[e]);
            f[2 * e + 1] = T::hi(v[e]);
        }
    }
    // elements c .. c + 7 of a row of n, zeros past it; WHOLE: n is a multiple of 8
    template <bool WHOLE = false>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        const uint16_t* p = static_cast<const uint16_t*>(row) + c;
        v = (u32x4_t){0, 0, 0, 0};
        if (WHOLE ? c < n : c + 8 <= n) {
            v = *reinterpret_cast<const chunk16_t*>(p);
        } else if (!WHOLE && c < n) {
            // (loads side by side: under a condition each, every one of them is waited for by itself)
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 7; ++e) h[e] = p[c + e < n ? e : 0];
            h[7] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = c + e < n ? h[e] : 0;
            v = (u32x4_t){h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6]};
        }
    }
    __device__ static __forceinline__ u32x4_t pack(const float (&f)[8])
    {
        return (u32x4_t){T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7])};
    }
    template <bool WHOLE = false>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        uint16_t* p = static_cast<uint16_t*>(row) + c;
        const u32x4_t w = pack(f);
        if (WHOLE ? c < n : c + 8 <= n) {
            *reinterpret_cast<chunk16_t*>(p) = w;
        } else if (!WHOLE && c < n) {
#pragma unroll
            for (int e = 0; e < 7; ++e)
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
    float v[8];
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v[e];
    }
    template <bool WHOLE = false>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        const float* p = static_cast<const float*>(row) + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        if (WHOLE ? c < n : c + 8 <= n) {
            const chunk32_t a = *reinterpret_cast<const chunk32_t*>(p), b = *reinterpret_cast<const chunk32_t*>(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = a[e];
                v[4 + e] = b[e];
            }
        } else if (!WHOLE && c < n) {
#pragma unroll
            for (int e = 0; e < 7; ++e) v[e] = p[c + e < n ? e : 0];
#pragma unroll
            for (int e = 0; e < 7; ++e) v[e] = c + e < n ? v[e] : 0.0f;
        }
    }
    template <bool WHOLE = false>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        float* p = static_cast<float*>(row) + c;
        if (WHOLE ? c < n : c + 8 <= n) {
            *reinterpret_cast<chunk32_t*>(p) = (chunk32_t){f[0], f[1], f[2], f[3]};
            *reinterpret_cast<chunk32_t*>(p + 4) = (chunk32_t){f[4], f[5], f[6], f[7]};
        } else if (!WHOLE && c < n) {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (c + e < n) p[e] = f[e];
        }
    }
};

inline int bytes_of(int hp_dtype) { return hp_dtype == MI8_F32 ? 4 : 2; }
inline bool float_type(int hp_dtype) { return hp_dtype == MI8_BF16 || hp_dtype == MI8_F16 || hp_dtype == MI8_F32; }

}  // namespace mi8
