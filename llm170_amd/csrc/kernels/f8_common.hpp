// Device helpers of the FP8 kernels: the scale of a block, and a lane's share of one, 32 elements in two runs of 16, as loaded and as e4m3.
#pragma once
#include "q8_common.hpp"

#define F8_ROWS 4  // as an element type: rows that are quantised already (W4A16_F8)

// The scale of a block from the bits of its largest magnitude: the least power of two that brings it to 448 (1.75 * 2^8) or below.  Zeros have the scale 0, infinity and
// NaN the scale NaN; `by` is what the elements are divided by, 1 there.
__device__ __forceinline__ float f8_step(unsigned mag, float& by) {
    const int e = max((int)(mag >> 23) - 8 + ((mag & 0x7fffffu) > 0x600000u ? 1 : 0), 1);  // biased; 1 is 2^-126
    const bool some = mag != 0 && mag < 0x7f800000u;
    const float s = q8_f32((unsigned)e << 23);
    by = some ? s : 1.f;
    return some ? s : mag == 0 ? 0.f : __builtin_nanf("");
}

// Largest of the eight lanes that share a block: neighbours, pairs, fours
__device__ __forceinline__ unsigned f8_block_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xb1, 0xf, 0xf, false));   // quad_perm 1 0 3 2
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4e, 0xf, 0xf, false));   // quad_perm 2 3 0 1
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, false));  // row_half_mirror
}

// Largest of 32 lanes
__device__ __forceinline__ unsigned f8_half_wave_max(unsigned v) {
    v = f8_block_max(v);
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, false));  // row_mirror
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // the even one's and the odd one's of each two rows of 16
    return max((unsigned)rows[0], (unsigned)rows[1]);
}

typedef short f8_pair_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));

// 16 consecutive elements as loaded
template <int T>
struct F8Run {
    static constexpr int WORDS = T == Q8_F32 ? 16 : 8;
    unsigned w[WORDS];
    // elements i .. i + 15 of a row; those from `left` on are zero and not read
    __device__ __forceinline__ void load(const char* row, int i, int left) {
        const char* const p = row + (size_t)(unsigned)i * (T == Q8_F32 ? 4 : 2);
        if (left >= 16) {
#pragma unroll
            for (int j = 0; j < WORDS / 4; j++) {
                const u4_any_t v = *reinterpret_cast<const u4_any_t*>(p + 16 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) w[4 * j + e] = v[e];
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < WORDS; e++) w[e] = 0;
        if (left <= 0) return;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (T == Q8_F32) {
                const unsigned v = *reinterpret_cast<const unsigned*>(p + 4 * min(e, left - 1));
                if (e < left) w[e % WORDS] = v;
            } else {
                const unsigned v = *reinterpret_cast<const uint16_t*>(p + 2 * min(e, left - 1));
                if (e < left) w[e / 2] |= v << (16 * (e & 1));
            }
        }
    }
    // the largest magnitude, as the bits of an f32; from infinity's on where one is infinity or NaN
    __device__ __forceinline__ unsigned most(unsigned m) const {
        if (T == Q8_F32) {
#pragma unroll
            for (int e = 0; e < WORDS; e++) m = max(m, w[e] & 0x7fffffffu);
            return m;
        }
        typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
        us2_t a = {0, 0};
#pragma unroll
        for (int e = 0; e < WORDS; e++) a = __builtin_elementwise_max(a, __builtin_bit_cast(us2_t, w[e] & 0x7fff7fffu));
        const unsigned b = max((unsigned)a[0], (unsigned)a[1]);
        return max(m, T == Q8_F16 ? __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(_Float16, (unsigned short)b)) : b << 16);
    }
    // as e4m3, divided by a power of two: exact quotients, rounded once
    __device__ __forceinline__ u4_t pack(float by, bool zero) const {
        u4_t o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f8_pair_t r = {0, 0};
            if (T == Q8_F32) {
                r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, q8_f32(w[(4 * i) % WORDS]), q8_f32(w[(4 * i + 1) % WORDS]), by, false);
                r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, q8_f32(w[(4 * i + 2) % WORDS]), q8_f32(w[(4 * i + 3) % WORDS]), by, true);
            } else {
                const unsigned lo = w[(2 * i) % WORDS], hi = w[(2 * i + 1) % WORDS];
                if (T == Q8_F16) {
                    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(h2_t, lo), by, false);
                    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(h2_t, hi), by, true);
                } else {
                    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf2_t, lo), by, false);
                    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf2_t, hi), by, true);
                }
            }
            o[i] = zero ? 0u : __builtin_bit_cast(unsigned, r);
        }
        return o;
    }
};

// Four f32 numbers as e4m3, byte e of the result is value e's
__device__ __forceinline__ unsigned f8_pack4(float a, float b, float c, float d, float by, bool zero) {
    f8_pair_t r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, by, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, by, true);
    return zero ? 0u : __builtin_bit_cast(unsigned, r);
}
