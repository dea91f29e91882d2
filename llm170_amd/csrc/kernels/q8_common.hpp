// Device helpers of the 8-bit kernels: the layout of quantised rows and weights, element types, quantisation of a value.
//
// Tiles ("T16x64"): 16 rows x 64 k of int8, 1 KiB: 64 chunks of 16 consecutive k, chunk c * 16 + r = row r, k = 16 c .. 16 c + 15
// (c = 0..3).  The 64 chunks in order are the operand of v_mfma_i32_16x16x64_i8 (lane l: row l % 16, k group l / 16), and a
// pair of them side by side that of v_mfma_i32_32x32x32_i8, so every operand load is one contiguous KiB or 256-byte runs of it.
// Tiles are ordered [row / 16][k / 64], an even number of k tiles per row block.  Weights are padded with zeros in both
// directions; the padding of quantised activations is never initialised: as k it meets zero weights, and whole-number products
// of garbage with zero are zero; as rows it gives results that nobody stores.
// Activations of few rows use tiles of R = 1 (one row) or 4 (two to four) instead of 16 rows: [row / R][k / 64][c][R] chunks.
#pragma once
#include "w4a16_common.hpp"

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i16_t __attribute__((ext_vector_type(16)));
// 16- and 8-byte accesses at element alignment: rows of odd length start anywhere
typedef unsigned u4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u2_any_t __attribute__((ext_vector_type(2), aligned(2)));

#define Q8_MAX_K 131071  // 128 * 128 * k stays below 2^31

#define Q8_F32 0  // element types (W4A16_F32 ..)
#define Q8_F16 1
#define Q8_BF16 2

// By value: a bit cast of an element of a vector in place reads element 0 (this compiler)
__device__ __forceinline__ float q8_f32(unsigned bits) { return __builtin_bit_cast(float, bits); }
__device__ __forceinline__ float q8_half(unsigned two, int which) { return (float)__builtin_bit_cast(h2_t, two)[which]; }
__device__ __forceinline__ float q8_bf16(unsigned bits) { return __builtin_bit_cast(float, bits << 16); }

// f32 -> bf16 bits, to nearest even; a NaN stays one
__device__ __forceinline__ unsigned q8_to_bf16(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v);
    return v != v ? 0x7fc0u : (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
}

// A 16-bit result.  The empty asm keeps the value a rounded f32 first, as in the separate kernels.
template <int T>
__device__ __forceinline__ unsigned q8_to_16(float v) {
    asm volatile("" : "+v"(v));
    return T == Q8_F16 ? (unsigned)__builtin_bit_cast(unsigned short, (_Float16)v) : q8_to_bf16(v);
}

template <int T>
__device__ __forceinline__ float q8_load1(const void* p, size_t i) {
    if (T == Q8_F32) return static_cast<const float*>(p)[i];
    if (T == Q8_F16) return (float)static_cast<const _Float16*>(p)[i];
    return q8_bf16(static_cast<const uint16_t*>(p)[i]);
}

// Sixteen consecutive elements from p[i]; those from `left` on are zero and not read.
template <int T>
__device__ __forceinline__ void q8_load16(const void* p, size_t i, int left, float (&v)[16]) {
    if (left >= 16) {
        if (T == Q8_F32) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u4_any_t w = *reinterpret_cast<const u4_any_t*>(static_cast<const float*>(p) + i + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * j + e] = q8_f32(w[e]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const u4_any_t w = *reinterpret_cast<const u4_any_t*>(static_cast<const uint16_t*>(p) + i + 8 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[8 * j + 2 * e] = T == Q8_F16 ? q8_half(w[e], 0) : q8_bf16(w[e] & 0xffffu);
                    v[8 * j + 2 * e + 1] = T == Q8_F16 ? q8_half(w[e], 1) : q8_f32(w[e] & 0xffff0000u);
                }
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = 0.f;
    if (left <= 0) return;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float w = q8_load1<T>(p, i + min(e, left - 1));
        if (e < left) v[e] = w;
    }
}

// |v| as an integer that orders as the magnitude does; infinity and NaN come out largest
__device__ __forceinline__ unsigned q8_mag(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// The size of a step from the largest magnitude of a row: fl32(max / 127), 0 for a row of (nearly) nothing (below the smallest
// normal number the quotients by it would be coarse), NaN for a row that holds infinity or NaN.
__device__ __forceinline__ float q8_step(unsigned mag) {
    if (mag >= 0x7f800000u) return __builtin_nanf("");
    const float s = __builtin_bit_cast(float, mag) / 127.0f;
    return s < 1.17549435e-38f ? 0.0f : s;
}

// The whole number nearest to x / s, halves to the even one, exactly: a candidate from the reciprocal is within one of it, its
// remainder x - q s is a multiple of the last place of s or of x and below 2^24 of them, so that the fused multiply-add gives it
// exactly, and it says on which side of a half x / s lies.  r = 1 / s (any rounding); s = 0 or NaN: r is 0 and q comes out 0.
__device__ __forceinline__ int q8_round(float x, float s, float r) {
    const float q = __builtin_rintf(x * r);
    const float d = __builtin_fmaf(-q, s, x), twice = 2.0f * __builtin_fabsf(d);
    const bool off = twice > s || (twice == s && ((int)q & 1));
    const float c = off ? q + __builtin_copysignf(1.0f, d) : q;
    return r == 0.f ? 0 : (int)c;
}

__device__ __forceinline__ float q8_recip(float s) { return s > 0.f ? 1.0f / s : 0.f; }  // NaN > 0 is false

// N values of a row quantised, byte e of the result is value e's (two's complement).  x * r + 128 is off by less than 2^-15: r and the sum
// are rounded once each, |x * r| <= 127.  Only where it lies within 1/20000 of a half (for sixteen values a lane one wave in ten) q8_round is asked.
template <int N>
__device__ __forceinline__ void q8_pack(const float (&w)[N], float step, float r, unsigned (&out)[N / 4]) {
    float far = 0.f, q[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        const float p = __builtin_fmaf(w[e], r, 128.0f);
        q[e] = __builtin_rintf(p);
        far = __builtin_fmaxf(far, __builtin_fabsf(p - q[e]));
    }
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        unsigned b = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) b = __builtin_amdgcn_cvt_pk_u8_f32(q[4 * i + e], e, b);
        out[i] = r == 0.f ? 0u : b ^ 0x80808080u;  // r = 0: nothing but zeros
    }
    if (__any(far > 0.49995f)) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            unsigned b = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) b |= ((unsigned)q8_round(w[4 * i + e], step, r) & 0xffu) << (8 * e);
            out[i] = b;
        }
    }
}

// Largest of one value per lane: rows of 16 by shifts, then across the rows, to lane 63
__device__ __forceinline__ unsigned q8_wave_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x111, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x112, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x114, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x118, 0xf, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x142, 0xa, 0xf, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x143, 0xc, 0xf, false));
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// Byte offset of chunk (row, 16 k from kc * 16) in a buffer of quantised rows with kt k tiles, tiles of R rows
__device__ __forceinline__ size_t q8_chunk_at(int row, int kc, int kt, int R) {
    return ((((size_t)(row / R) * kt + (kc >> 2)) * 4 + (kc & 3)) * R + row % R) * 16;
}
