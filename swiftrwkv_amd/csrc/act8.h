// Device helpers of the training-side operators (norm.hip, linear.hip): rows
// in chunks of 8 values of any element type and alignment, and the 8-bit
// activation checkpoint (MXINT8 of the OCP Microscaling Formats v1.0
// specification, written from its definition).
//
// A checkpoint of rows [N, D] is codes int8 [N, Dp], Dp = D rounded up to 32,
// and one scale byte per 32 codes, [N, Dp/32].  With e = floor(log2 amax) of
// a group (amax the largest magnitude of its 32 values), the scale byte is
// e + 127 and code = clamp(rint(x·2^(6-e)), ±127): the value it stands for is
// code·2^(e-6).  The step is a power of two, so x·2^(6-e) and code·2^(e-6)
// are exact: a code depends on no rounding but rint's own (half a step, 2^-7
// of 2^e; up to one step where |x| > 127.5 steps clamps, which keeps the
// largest finite values from restoring as infinity), and a restored value is
// exact in bf16, whose 8 significant bits hold 7-bit codes.  Scale bytes below
// 7 are raised to 7, so steps are normal fp32 numbers (groups under 2^-120
// restore with that step); 255 marks a group that held an infinity or a NaN:
// all of it restores as NaN.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

namespace rwkv_train {

constexpr int GROUP = 32;   // values per scale

__host__ __device__ inline int64_t padded(int64_t d) { return (d + GROUP - 1) / GROUP * GROUP; }

template <typename T>
__device__ __forceinline__ float to_f(T x) {
    return (float)x;
}

// Eight values from p, valid of them in range (the others 0).  Whole chunks
// load as 16-byte pieces at whatever alignment p has (gfx950 takes any).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
    if (valid >= 8) {
        T raw[8];
        __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f(p[i]) : 0.0f;
    }
}

// Eight values as loaded, to be converted later: a row that is on its way
// while another is worked on.
template <typename T>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int valid) {
        if (valid >= 8) {
            __builtin_memcpy(q, p, sizeof(q));
        } else {
            T t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = i < valid ? p[i] : (T)0.0f;
            __builtin_memcpy(q, t, sizeof(q));
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        T t[8];
        __builtin_memcpy(t, q, sizeof(q));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(t[i]);
    }
};

// Stores the first `valid` of eight values, each rounded once to T.
template <typename T>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[8]) {
    if (valid >= 8) {
        T raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = (T)v[i];
        __builtin_memcpy(p, raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}

// The step 2^(scale - 133) of a scale byte; NaN for 255.
__device__ __forceinline__ float step_of(uint32_t scale) {
    return __builtin_bit_cast(float, scale == 255u ? 0x7fc00000u : (scale - 6u) << 23);
}

// Scale byte of a group whose largest magnitude has the bits amax (255:
// infinity or NaN, whose patterns are the largest).
__device__ __forceinline__ uint32_t scale_of(uint32_t amax) { return max(amax >> 23, 7u); }

// Bits of the largest magnitude of eight values.
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    return m;
}

// The low bytes of four dwords.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// Encodes a group's share of four neighbouring lanes (8 values each, lanes
// 4q .. 4q+3 in column order): returns the lane's eight codes and the group's
// scale byte.  Every lane of the quad must be active.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t& scale) {
    uint32_t m = amax8(v);
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    scale = scale_of(m);
    const float inv = __builtin_bit_cast(float, (260u - min(scale, 254u)) << 23);   // 2^(133 - scale)
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)   // 1.5·2^23 rounds to an integer, in the low byte as two's complement
        w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(v[i] * inv, -127.0f, 127.0f) + 12582912.0f);
    const bool bad = scale == 255u;
    return make_uint2(bad ? 0u : low_bytes(w[0], w[1], w[2], w[3]), bad ? 0u : low_bytes(w[4], w[5], w[6], w[7]));
}

// The eight values of codes c with the group's scale byte.
__device__ __forceinline__ void decode8(uint2 c, uint32_t scale, float (&v)[8]) {
    const float step = step_of(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = i < 4 ? c.x : c.y;
        v[i] = (float)(int)(int8_t)(w >> (8 * (i & 3))) * step;
    }
}

}  // namespace rwkv_train
