// Device helpers of the kernels that go over rows of logits: a lane's 64 bytes of a wave's stage, orders and maxima.
#pragma once
#include "q8_common.hpp"

#define SCORE_LOG2E 1.44269504088896341f

// Lane 63 of the result combines all 64: rows of 16 by shifts, then across the rows
template <int CTRL, int ROWS>
__device__ __forceinline__ float score_dpp(float old, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float score_wave_max(float v) {  // NaN where a lane has one
    v = __builtin_elementwise_maximum(v, score_dpp<0x111, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x112, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x114, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x118, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x142, 0xa>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x143, 0xc>(v, v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Larger for the larger value; NaN above all, -0 as 0
__device__ __forceinline__ unsigned score_order(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);
    return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// 64 bytes of raw elements per lane: E of them, element e is index at(e) of the stage
template <int T>
struct ScoreChunk {
    static constexpr int N = 4, PER = T == Q8_F32 ? 4 : 8, SIZE = T == Q8_F32 ? 4 : 2, E = N * PER, STAGE = 64 * E;
    u4_t w[N];

    static __device__ __forceinline__ int at(int lane, int e) { return (e / PER) * (PER * 64) + lane * PER + e % PER; }
    // p: the stage's first element (uniform), n: the elements that there are from it on; those behind them read as -infinity
    __device__ __forceinline__ void load(const char* p, unsigned n, int lane) {
        if (n >= STAGE) {
#pragma unroll
            for (int j = 0; j < N; j++) w[j] = *reinterpret_cast<const u4_any_t*>(p + lane * 16 + j * 1024);
            return;
        }
        const unsigned none = T == Q8_F32 ? 0xff800000u : T == Q8_F16 ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int j = 0; j < N; j++) {
            w[j] = (u4_t){none, none, none, none};
            if (at(lane, j * PER) + PER <= (int)n) w[j] = *reinterpret_cast<const u4_any_t*>(p + lane * 16 + j * 1024);
        }
        // the 16 bytes of one lane that the end lies in
        const int left = (int)n % PER, vec = (int)n / PER;
        if (left == 0) return;
        if (lane == vec % 64) {
            u4_t t = {none, none, none, none};
#pragma unroll
            for (int d = 0; d < PER - 1; d++) {
                const unsigned at_d = (n - left + min(d, left - 1)) * SIZE;
                if (T == Q8_F32) {
                    const unsigned v = *reinterpret_cast<const unsigned*>(p + at_d);
                    if (d < left) t[d] = v;
                } else {
                    const unsigned v = *reinterpret_cast<const uint16_t*>(p + at_d);
                    if (d < left) t[d / 2] = d & 1 ? (t[d / 2] & 0xffffu) | v << 16 : (t[d / 2] & 0xffff0000u) | v;
                }
            }
#pragma unroll
            for (int j = 0; j < N; j++)
                if (j == vec / 64) w[j] = t;
        }
    }
    // Forgets the values that were computed from the raw elements, which else stay in registers from one use to the next
    __device__ __forceinline__ void fresh() {
#pragma unroll
        for (int i = 0; i < N * 4; i++) {
            unsigned d = w[i / 4][i % 4];
            asm volatile("" : "+v"(d));
            w[i / 4][i % 4] = d;
        }
    }
    __device__ __forceinline__ float value(int e) const {
        const unsigned d = w[e / PER][T == Q8_F32 ? e % PER : e % PER / 2];
        if (T == Q8_F32) return q8_f32(d);
        if (T == Q8_F16) return q8_half(d, e & 1);
        return (e & 1) ? q8_f32(d & 0xffff0000u) : q8_bf16(d & 0xffffu);
    }
    // value(e) * L - r, one rounding; an f16 enters the multiply-add as it is
    __device__ __forceinline__ float scaled(int e, float r) const {
        if (T != Q8_F16) return __builtin_fmaf(value(e), SCORE_LOG2E, -r);
        float d;
        const unsigned h = w[e / PER][e % PER / 2];
        const float l = SCORE_LOG2E;
        if (e & 1) asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "s"(l), "v"(r));
        else asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "s"(l), "v"(r));
        return d;
    }
    // value(e) - m; an f16 enters the subtraction as it is
    __device__ __forceinline__ float minus(int e, float m) const {
        if (T != Q8_F16) return value(e) - m;
        float d;
        const unsigned h = w[e / PER][e % PER / 2];
        if (e & 1) asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(m));
        else asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(m));
        return d;
    }
    // the largest and the smallest (NaN if there is one); f16 two at a time
    __device__ __forceinline__ void extremes(float& most, float& least) const {
        if (T == Q8_F16) {
            auto pair = [&](int i) { const unsigned d = w[i / 4][i % 4]; return __builtin_bit_cast(h2_t, d); };
            h2_t a = pair(0), b = pair(0);
#pragma unroll
            for (int i = 1; i < E / 2; i++) {
                a = __builtin_elementwise_maximum(a, pair(i));
                b = __builtin_elementwise_minimum(b, pair(i));
            }
            most = __builtin_elementwise_maximum((float)a[0], (float)a[1]);
            least = __builtin_elementwise_minimum((float)b[0], (float)b[1]);
        } else {
            most = __builtin_elementwise_maximum(value(0), value(1));
            least = __builtin_elementwise_minimum(value(0), value(1));
#pragma unroll
            for (int e = 2; e < E; e += 2) {
                most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, value(e)), value(e + 1));
                least = __builtin_elementwise_minimum(__builtin_elementwise_minimum(least, value(e)), value(e + 1));
            }
        }
    }
};
