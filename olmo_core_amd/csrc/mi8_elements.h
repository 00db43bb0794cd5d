// Eight consecutive elements of a row of bf16, float16 or float32, in float32 registers.
//
// A lane's eight elements are one access of 16 bytes (two in float32) at any address: gfx950 serves global loads and stores at the alignment of the element, so
// rows of odd length need no other kernel, only their last chunk an element at a time (16-bit elements one by one instead: gradient of the epilogue,
// 1537 x 2771, 48 us).  Rows known to have eight elements and more (LONG) take the last chunk as the row's last eight, moved down to their places, and
// store it in up to three pieces: fewer registers and accesses.
#pragma once
#include "mi8_half.h"

namespace mi8 {

typedef uint32_t chunk16_t __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's alignment
typedef uint32_t chunk8_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t chunk4_t __attribute__((aligned(2)));
typedef float chunk32_t __attribute__((ext_vector_type(4), aligned(4)));
typedef float chunk32h_t __attribute__((ext_vector_type(2), aligned(4)));

// (a choice between two elements of an array by itself is one between their addresses, and puts the array into memory)
__device__ __forceinline__ float pick(int c, float a, float b) { return c ? a : b; }

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
    // elements c .. c + 7 of a row of n, zeros past it; WHOLE: n is a multiple of 8; LONG: n is 8 or more, or 0
    template <bool WHOLE = false, bool LONG = false>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        const uint16_t* p = static_cast<const uint16_t*>(row) + c;
        v = (u32x4_t){0, 0, 0, 0};
        if (!WHOLE && LONG) {
            if (c >= n) return;
            const int past = max(c + 8 - n, 0);
            v = *reinterpret_cast<const chunk16_t*>(p - past);
            if (past & 4) v = (u32x4_t){v[2], v[3], 0, 0};
            if (past & 2) v = (u32x4_t){v[1], v[2], v[3], 0};
            if (past & 1) v = (u32x4_t){v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
            return;
        }
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
    template <bool WHOLE = false, bool LONG = false>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        uint16_t* p = static_cast<uint16_t*>(row) + c;
        const u32x4_t w = pack(f);
        if (WHOLE ? c < n : c + 8 <= n) {
            *reinterpret_cast<chunk16_t*>(p) = w;
        } else if (!WHOLE && LONG && c < n) {
            const int some = n - c;
            u32x4_t x = w;
            if (some & 4) {
                *reinterpret_cast<chunk8_t*>(p) = (chunk8_t){x[0], x[1]};
                x = (u32x4_t){x[2], x[3], 0, 0};
            }
            if (some & 2) {
                *reinterpret_cast<chunk4_t*>(p + (some & 4)) = x[0];
                x[0] = x[1];
            }
            if (some & 1) p[some & 6] = (uint16_t)x[0];
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
    template <bool WHOLE = false, bool LONG = false>
    __device__ __forceinline__ void load(const void* row, int c, int n)
    {
        const float* p = static_cast<const float*>(row) + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        if (!WHOLE && LONG) {
            if (c >= n) return;
            const int past = max(c + 8 - n, 0);
            const chunk32_t a = *reinterpret_cast<const chunk32_t*>(p - past), b = *reinterpret_cast<const chunk32_t*>(p - past + 4);
            const float x[12] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], 0.0f, 0.0f, 0.0f, 0.0f};
            float y[10];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = pick(past & 4, x[e + 4], x[e]);
            y[8] = y[9] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = pick(past & 2, e < 6 ? v[(e + 2) & 7] : 0.0f, v[e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = pick(past & 1, y[e + 1], y[e]);
            return;
        }
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
    template <bool WHOLE = false, bool LONG = false>
    __device__ static __forceinline__ void store(void* row, int c, int n, const float (&f)[8])
    {
        float* p = static_cast<float*>(row) + c;
        if (WHOLE ? c < n : c + 8 <= n) {
            *reinterpret_cast<chunk32_t*>(p) = (chunk32_t){f[0], f[1], f[2], f[3]};
            *reinterpret_cast<chunk32_t*>(p + 4) = (chunk32_t){f[4], f[5], f[6], f[7]};
        } else if (!WHOLE && LONG && c < n) {
            const int some = n - c;
            chunk32_t w = {f[0], f[1], f[2], f[3]};
            const chunk32_t high = {f[4], f[5], f[6], f[7]};
            if (some & 4) {
                *reinterpret_cast<chunk32_t*>(p) = w;
                w = high;
            }
            if (some & 2) {
                *reinterpret_cast<chunk32h_t*>(p + (some & 4)) = (chunk32h_t){w[0], w[1]};
                w = (chunk32_t){w[2], w[3], 0.0f, 0.0f};
            }
            if (some & 1) p[some & 6] = w[0];
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
