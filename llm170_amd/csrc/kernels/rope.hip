// Queries and keys between a layer's QKV projection and its attention: every head's RMS norm and the rotation of its first `rot` elements by the row's
// position, in one pass.  v <- v / sqrt(mean v^2 + eps) * w (w per element, one set for queries and one for keys, where there is one), then for every pair
// (a, b) of the rotated part and its angle, position * frequency, (a cos - b sin, b cos + a sin), cosine and sine times `amp`.  Pairs are (c, c + rot / 2) or
// (2 c, 2 c + 1).
//
// Each element is read and written once, which is what bounds many rows.  A wave takes one row and goes over its heads, as many at a time as its lanes hold: a unit of
// VEC pairs (or 2 VEC elements behind the rotated part) to a lane, G lanes to a head.  The row's cosines and sines are computed once, a pair to a lane, and kept in LDS.  Angles
// are reduced to a part of a turn in 64 bits: at position 10^6 an f32 product is off by 0.06.  Few rows: a row's heads go to several waves.
#include "q8_common.hpp"

#define ROPE_MAX_DIM 1024  // elements of a head
#define ROPE_WAVES 4

// N consecutive elements of type T, as loaded
template <int T, int N>
struct RopeRaw {
    static constexpr int BYTES = N * (T == Q8_F32 ? 4 : 2), WORDS = (BYTES + 3) / 4;
    unsigned w[WORDS];
    __device__ __forceinline__ void load(const void* p, size_t i) {
        const char* const at = static_cast<const char*>(p) + i * (T == Q8_F32 ? 4 : 2);
        if (BYTES >= 16) {
#pragma unroll
            for (int j = 0; j < BYTES / 16; j++) {
                const u4_any_t v = *reinterpret_cast<const u4_any_t*>(at + 16 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) w[(4 * j + e) % WORDS] = v[e];
            }
        } else if (BYTES == 8) {
            const u2_any_t v = *reinterpret_cast<const u2_any_t*>(at);
            w[0] = v[0];
            w[1 % WORDS] = v[1];
        } else if (BYTES == 4) {
            typedef unsigned u1_any_t __attribute__((aligned(2)));
            w[0] = *reinterpret_cast<const u1_any_t*>(at);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(at);
        }
    }
    __device__ __forceinline__ float get(int e) const {
        const unsigned d = w[T == Q8_F32 ? e : e / 2];
        if (T == Q8_F32) return q8_f32(d);
        if (T == Q8_F16) return q8_half(d, e & 1);
        return (e & 1) ? q8_f32(d & 0xffff0000u) : q8_bf16(d & 0xffffu);
    }
};

template <int T, int N>
__device__ __forceinline__ void rope_store(void* y, size_t i, const float* v) {
    if (T == Q8_F32) {
        float* const p = static_cast<float*>(y) + i;
        if (N % 4 == 0) {
#pragma unroll
            for (int j = 0; j < N / 4; j++)
                *reinterpret_cast<u4_any_t*>(p + 4 * j) = (u4_any_t){__builtin_bit_cast(unsigned, v[4 * j]), __builtin_bit_cast(unsigned, v[4 * j + 1]),
                                                                     __builtin_bit_cast(unsigned, v[4 * j + 2]), __builtin_bit_cast(unsigned, v[4 * j + 3])};
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) p[e] = v[e];
        }
        return;
    }
    uint16_t* const p = static_cast<uint16_t*>(y) + i;
    unsigned h[N];
#pragma unroll
    for (int e = 0; e < N; e++) h[e] = q8_to_16<T>(v[e]);
    if (N % 8 == 0) {
#pragma unroll
        for (int j = 0; j < N / 8; j++)
            *reinterpret_cast<u4_any_t*>(p + 8 * j) = (u4_any_t){h[8 * j] | h[8 * j + 1] << 16, h[8 * j + 2] | h[8 * j + 3] << 16, h[8 * j + 4] | h[8 * j + 5] << 16,
                                                                 h[8 * j + 6] | h[8 * j + 7] << 16};
    } else if (N == 2) {
        typedef unsigned u1_any_t __attribute__((aligned(2)));
        *reinterpret_cast<u1_any_t*>(p) = h[0] | h[1 % N] << 16;
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = (uint16_t)h[e];
    }
}

// lg: log2 of the lanes to a head.  x and the results may be the same rows, so nothing is said to be restricted: a head is read before it is written, element by element
// by the same lane.
template <int T, int VEC, bool IL>
__device__ __forceinline__ void rope_body(const void* x, size_t ldx, int t, int nq, int nk, int dim, int rot, const float* qw, const float* kw,
                                          float eps, const int* pos, const double* freqs, float amp, void* q, size_t ldq, void* k, size_t ldk, int y_type, int lg,
                                          int splits) {
    constexpr int NU = ROPE_MAX_DIM / (2 * VEC * 64);  // units of a lane
    __shared__ float table[ROPE_WAVES][2][ROPE_MAX_DIM / 2];  // cosines, sines
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned id = blockIdx.x * ROPE_WAVES + wave;
    const int row = (int)(id / (unsigned)splits), split = (int)(id - (unsigned)row * splits);
    if (row >= t) return;
    const int g = 1 << lg, hp = 64 >> lg, in = lane & (g - 1), half = rot >> 1, turning = half / VEC, units = turning + (dim - rot + 2 * VEC - 1) / (2 * VEC);
    const int q_passes = (nq + hp - 1) / hp, passes = q_passes + (nk + hp - 1) / hp;
    // where the two runs of a unit begin
    auto first = [&](int u) { return u < turning ? u * VEC * (IL ? 2 : 1) : rot + (u - turning) * 2 * VEC; };
    auto second = [&](int u) { return u < turning && !IL ? half + u * VEC : first(u) + VEC; };  // behind an odd head's end there may be none
    RopeRaw<T, VEC> raw[NU][2];
    auto head_of = [&](int pass) { return (pass < q_passes ? pass : pass - q_passes) * hp + (lane >> lg); };  // among the queries or the keys
    auto load = [&](int pass) {
        const bool key = pass >= q_passes;
        const int head = head_of(pass);
        if (head >= (key ? nk : nq)) return;
        const size_t at = (size_t)row * ldx + (size_t)((key ? nq : 0) + head) * dim;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = in + i * g;
            if (i * g >= units) break;  // uniform
            if (u >= units) continue;
            raw[i][0].load(x, at + first(u));
            if (VEC > 1 || second(u) < dim) raw[i][1].load(x, at + second(u));
        }
    };
    load(split);
    float cs[NU][VEC], sn[NU][VEC];
    if (rot > 0) {
        const double p = (double)pos[row] * 0.15915494309189533577;  // turns
        for (int c = lane; c < half; c += 64) {
            const double turns = p * freqs[c];
            float s, co;
            sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &co);
            table[wave][0][c] = co * amp;
            table[wave][1][c] = s * amp;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // one wave's table: its instructions are in order
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (i * g >= units) break;
            const int u = min(in + i * g, turning - 1);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                cs[i][e] = table[wave][0][u * VEC + e];
                sn[i][e] = table[wave][1][u * VEC + e];
            }
        }
    }
    float w[NU][2 * VEC];
    int have = -1;  // whose weights these are
    const float inv_dim = 1.0f / (float)dim;
    for (int pass = split; pass < passes; pass += splits) {
        const bool key = pass >= q_passes;
        const int head = head_of(pass);
        const bool mine = head < (key ? nk : nq);
        const float* const weight = key ? kw : qw;
        if (weight && have != (int)key) {
            have = (int)key;
#pragma unroll
            for (int i = 0; i < NU; i++) {
                const int u = in + i * g;
                if (i * g >= units) break;
                if (u >= units) continue;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    w[i][e] = weight[first(u) + e];
                    w[i][VEC + e] = VEC > 1 || second(u) < dim ? weight[second(u) + e] : 0.f;
                }
            }
        }
        float v[NU][2 * VEC];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (i * g >= units) break;
            const int u = in + i * g;
            const bool one = mine && u < units, two = one && (VEC > 1 || second(u) < dim);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                v[i][e] = one ? raw[i][0].get(e) : 0.f;
                v[i][VEC + e] = two ? raw[i][1].get(e) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) ss = __builtin_fmaf(v[i][e], v[i][e], ss);
        }
        if (pass + splits < passes) load(pass + splits);
        if (weight) {
            for (int d = 1; d < g; d <<= 1) ss += __shfl_xor(ss, d);
            const float inv = 1.0f / sqrtf(__builtin_fmaf(ss, inv_dim, eps));
#pragma unroll
            for (int i = 0; i < NU; i++) {
                if (i * g >= units) break;
#pragma unroll
                for (int e = 0; e < 2 * VEC; e++) v[i][e] = v[i][e] * inv * w[i][e];
            }
        }
        if (!mine) continue;
        void* const out = key ? k : q;
        const size_t at = (size_t)row * (key ? ldk : ldq) + (size_t)head * dim;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (i * g >= units) break;
            const int u = in + i * g;
            if (u >= units) continue;
            if (u < turning) {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    constexpr int STEP = IL ? 2 : 1;
                    float &a = v[i][STEP * e], &b = v[i][IL ? 2 * e + 1 : VEC + e];
                    const float turned = __builtin_fmaf(-b, sn[i][e], a * cs[i][e]);
                    b = __builtin_fmaf(a, sn[i][e], b * cs[i][e]);
                    a = turned;
                }
            }
            auto store = [&](auto type) {
                constexpr int Y = decltype(type)::value;
                rope_store<Y, VEC>(out, at + first(u), v[i]);
                if (VEC > 1 || second(u) < dim) rope_store<Y, VEC>(out, at + second(u), v[i] + VEC);
            };
            if (y_type == Q8_F32) store(w8_type<Q8_F32>{});
            else if (y_type == Q8_F16) store(w8_type<Q8_F16>{});
            else store(w8_type<Q8_BF16>{});
        }
    }
}

#define ROPE_KERNEL(NAME, T, VEC, IL)                                                                                              \
    extern "C" __global__ __launch_bounds__(ROPE_WAVES * 64) void NAME(const void* x, size_t ldx, int t, int nq, int nk, int dim, int rot, const float* qw, \
                                                                       const float* kw, float eps, const int* pos, const double* freqs, float amp, void* q, \
                                                                       size_t ldq, void* k, size_t ldk, int y_type, int lg, int splits) {      \
        rope_body<T, VEC, IL>(x, ldx, t, nq, nk, dim, rot, qw, kw, eps, pos, freqs, amp, q, ldq, k, ldk, y_type, lg, splits);       \
    }
#define ROPE_KERNELS(SUFFIX, VEC, IL)                              \
    ROPE_KERNEL(w4a16_qk_norm_rope_f32##SUFFIX, Q8_F32, VEC, IL)   \
    ROPE_KERNEL(w4a16_qk_norm_rope_f16##SUFFIX, Q8_F16, VEC, IL)   \
    ROPE_KERNEL(w4a16_qk_norm_rope_bf16##SUFFIX, Q8_BF16, VEC, IL)
ROPE_KERNELS(_v8, 8, false)
ROPE_KERNELS(_v2, 2, false)
ROPE_KERNELS(_v1, 1, false)
ROPE_KERNELS(_v8_il, 8, true)
ROPE_KERNELS(_v2_il, 2, true)
ROPE_KERNELS(_v1_il, 1, true)
