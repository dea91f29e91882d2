// W8A8 linears:  y[m][n] = (sum_k q[m][k] w[n][k]) * s[m] * ws[n],  q and w int8 in tiles (q8_common.hpp), sums in 32-bit whole
// numbers (exact: k <= 131071), one f32 scale per row of either.  Gated form: rows 0..n/2 of w are a gate, the rest its values,
// y[m][c] = act(gate) * value, [t][n/2].
#include "q8_common.hpp"

// y[at .. at + 3] (those below `left`) as f32, f16 or bf16
__device__ __forceinline__ void w8_store4(void* __restrict__ y, size_t at, int left, const float (&v)[4], int y_type) {
    if (y_type == Q8_F32) {
        float* const p = static_cast<float*>(y) + at;
        if (left >= 4) {
            u4_any_t o;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_bit_cast(unsigned, v[i]);
            *reinterpret_cast<u4_any_t*>(p) = o;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < left) p[i] = v[i];
        }
        return;
    }
    unsigned h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = y_type == Q8_F16 ? q8_to_16<Q8_F16>(v[i]) : q8_to_16<Q8_BF16>(v[i]);
    uint16_t* const p = static_cast<uint16_t*>(y) + at;
    if (left >= 4) {
        u2_any_t o;
        o[0] = h[0] | h[1] << 16;
        o[1] = h[2] | h[3] << 16;
        *reinterpret_cast<u2_any_t*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = (uint16_t)h[i];
    }
}

// ------------------------------------------------------------------------------------------------ up to 64 rows
// The weight stream bounds these launches.  A workgroup's waves take consecutive runs of a k slice of the same RB row blocks (16
// outputs each); the weights arrive as whole tiles straight in registers, DEPTH of them in flight per row block, meet TT tiles of 16
// activation rows (from the L2), and the waves' sums are added in LDS: whole numbers, so in any order the same.  Where there are too
// few row blocks for the chip, slices of k go to several workgroups (gridDim.y of them): each leaves its sums in the workspace and
// draws a ticket of its row blocks, the last one adds them.
typedef unsigned long long w8_pair_t;

template <int RB, int TT, bool GLU>
__device__ __forceinline__ void skinny_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                            const float* __restrict__ xs, void* __restrict__ y, int n, int kt, int t, int R, int y_type, int act, int W,
                                            int nks, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int DEPTH = RB * TT == 1 ? 8 : RB + TT <= 4 ? 4 : RB + TT <= 6 ? 3 : 2, TILES = RB * TT;
    __shared__ int sums[TILES][4][64];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_blocks = (n + 15) >> 4, half_rb = GLU ? row_blocks >> 1 : 0;
    // row block of slot i: gated, slots 2j and 2j + 1 are a gate's and its values'
    auto block_of = [&](int i) { return GLU ? blockIdx.x * (RB / 2) + i / 2 + (i & 1 ? half_rb : 0) : blockIdx.x * RB + i; };
    const int last = (GLU ? half_rb : row_blocks) - 1;
    const char* wp[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) {
        int b = block_of(i);
        if (GLU) b = min(b - (i & 1 ? half_rb : 0), last) + (i & 1 ? half_rb : 0);  // slots past the end read the last block, not stored
        else b = min(b, last);
        wp[i] = wt + (size_t)b * kt * 1024 + lane * 16;
    }
    const int tok = lane & 15, kg = lane >> 4;
    // activations: tiles of R rows, [k tile][kg][R] chunks
    const char* const xp = xq + ((size_t)kg * R + tok % R) * 16;
    const size_t x_tile = (size_t)R * 64, x_block = x_tile * kt;

    const int runs = nks * W, run = blockIdx.y * W + wave;
    const int lo = (int)((long long)kt * run / runs), hi = (int)((long long)kt * (run + 1) / runs);
    i4_t acc[RB][TT];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = (i4_t){0, 0, 0, 0};
    i4_t wv[DEPTH][RB], xv[DEPTH][TT];
    auto load = [&](int d, int k) {
#pragma unroll
        for (int i = 0; i < RB; i++) wv[d][i] = __builtin_nontemporal_load(reinterpret_cast<const i4_t*>(wp[i] + (size_t)k * 1024));
#pragma unroll
        for (int j = 0; j < TT; j++) xv[d][j] = *reinterpret_cast<const i4_t*>(xp + j * x_block + k * x_tile);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (lo + d < hi) load(d, lo + d);
    if (W > 1) {
        for (int i = threadIdx.x; i < TILES * 256; i += W * 64) (&sums[0][0][0])[i] = 0;
        __syncthreads();
    }
    for (int k = lo; k < hi; k += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            if (k + d < hi) {
#pragma unroll
                for (int i = 0; i < RB; i++)
#pragma unroll
                    for (int j = 0; j < TT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[d][i], xv[d][j], acc[i][j], 0, 0, 0);
                if (k + d + DEPTH < hi) load(d, k + d + DEPTH);
            }
        }
    }
    if (W > 1) {
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < TT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    __hip_atomic_fetch_add(&sums[i * TT + j][e][lane], acc[i][j][e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
    }
    // A wave finishes every W-th tile (gated: a gate and its values)
    auto total = [&](int tile) {
        i4_t v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = sums[tile][e][lane];
        return v;
    };
    constexpr int U = GLU ? RB / 2 : RB;
    const size_t slice = (size_t)gridDim.x * (TILES * 128);  // pairs of sums per k slice
    w8_pair_t* const mine = part + (size_t)blockIdx.x * (TILES * 128) + lane;
    if (nks > 1) {
        // Device-scope stores, complete before the ticket is drawn; device-scope loads behind the barrier that follows the ticket's return.
        // Neither is served from a cache that is not coherent.
#pragma unroll
        for (int u = 0; u < TILES; u++) {
            if (u % W != wave || (u % TT) * 16 + tok >= t) continue;
            const i4_t v = W > 1 ? total(u) : acc[u / TT][u % TT];
            w8_pair_t* const p = mine + blockIdx.y * slice + u * 128;
            __hip_atomic_store(p, (w8_pair_t)(unsigned)v[1] << 32 | (unsigned)v[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(p + 64, (w8_pair_t)(unsigned)v[3] << 32 | (unsigned)v[2], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) last_one = __hip_atomic_fetch_add(tickets + blockIdx.x, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nks - 1;
        __syncthreads();
        if (!last_one) return;
        if (threadIdx.x == 0) __hip_atomic_store(tickets + blockIdx.x, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    }
#pragma unroll
    for (int u = 0; u < U * TT; u++) {
        if (u % W != wave) continue;  // uniform for the wave
        const int i = GLU ? u / TT * 2 : u / TT, j = u % TT;
        const int b = block_of(i), m = j * 16 + tok, c = b * 16 + kg * 4;
        if (b > last || m >= t) continue;
        auto sum_of = [&](int i_) {
            if (nks == 1) return W > 1 ? total(i_ * TT + j) : acc[i_][j];
            i4_t v = {0, 0, 0, 0};
            const w8_pair_t* p = mine + (i_ * TT + j) * 128;
#pragma unroll 4
            for (int s = 0; s < nks; s++, p += slice) {
                const w8_pair_t a = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const w8_pair_t d = __hip_atomic_load(p + 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                v += (i4_t){(int)a, (int)(a >> 32), (int)d, (int)(d >> 32)};
            }
            return v;
        };
        const i4_t sum = sum_of(i), sum_up = GLU ? sum_of(i + 1) : sum;
        const float sx = xs[m];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = (float)sum[e] * sx * ws[c + e];
            if (GLU) v[e] = w4_act_mul(v[e], (float)sum_up[e] * sx * ws[c + half_rb * 16 + e], act);
        }
        const int out_n = GLU ? n >> 1 : n;
        w8_store4(y, (size_t)m * out_n + c, out_n - c, v, y_type);
    }
}

#define W8_SKINNY(NAME, RB, TT, GLU, THREADS)                                                                                     \
    extern "C" __global__ __launch_bounds__(THREADS) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                               int kt, int t, int R, int y_type, int act, int waves, int nks, w8_pair_t* part,   \
                                                               int* tickets) {                                                    \
        skinny_body<RB, TT, GLU>(wt, ws, xq, xs, y, n, kt, t, R, y_type, act, waves, nks, part, tickets);                         \
    }
#define W8_SKINNY_T(NAME, RB, GLU, SUFFIX)                \
    W8_SKINNY(NAME##_t1##SUFFIX, RB, 1, GLU, 512)         \
    W8_SKINNY(NAME##_t2##SUFFIX, RB, 2, GLU, 512)         \
    W8_SKINNY(NAME##_t3##SUFFIX, RB, 3, GLU, 512)         \
    W8_SKINNY(NAME##_t4##SUFFIX, RB, 4, GLU, 512)
W8_SKINNY_T(w4a16_w8a8_skinny_r1, 1, false, )
W8_SKINNY_T(w4a16_w8a8_skinny_r2, 2, false, )
W8_SKINNY_T(w4a16_w8a8_skinny_r4, 4, false, )
W8_SKINNY_T(w4a16_w8a8_skinny_r2, 2, true, _glu)
W8_SKINNY_T(w4a16_w8a8_skinny_r4, 4, true, _glu)

// ------------------------------------------------------------------------------------------------ tiles, any number of rows
// Block tile 32 MI rows x 256 columns, four waves along n, wave tile 32 MI x 64 on v_mfma_i32_32x32x32_i8.  Activations go
// through LDS by DMA, 128 k a stage, two stages; weights straight into registers, a stage ahead.
#define W8_KS 128
template <int MI, bool GLU>
__device__ __forceinline__ void tiled_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                           const float* __restrict__ xs, void* __restrict__ y, int n, int kt, int t, int y_type, int act) {
    extern __shared__ char lds[];
    constexpr int BM = 32 * MI, STAGE = BM * W8_KS, NA = STAGE / 4096;  // DMA loads per wave and stage
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nl = lane & 31, kh = lane >> 5;
    const int out_n = GLU ? n >> 1 : n, half_rb = GLU ? n >> 5 : 0, row_blocks = (n + 15) >> 4;
    constexpr int BN = GLU ? 128 : 256;
    // Block tiles: every XCD takes a consecutive eighth of them, bands of eight tile rows, in a band m fastest
    const int tiles_m = (t + BM - 1) / BM, tiles_n = (out_n + BN - 1) / BN;
    const unsigned work = (unsigned)tiles_m * (unsigned)tiles_n, xcd = blockIdx.x & 7;
    const unsigned at = (unsigned)((unsigned long long)work * xcd / 8) + (blockIdx.x >> 3);
    if (at >= (unsigned)((unsigned long long)work * (xcd + 1) / 8)) return;
    const unsigned band = at / (8u * tiles_n), in_band = at - band * 8u * tiles_n;
    const unsigned rows = min(8u, (unsigned)tiles_m - band * 8u);
    const int tn = (int)(in_band / rows), tm = (int)(band * 8u + in_band - tn * rows);
    const int m0 = tm * BM, n0 = tn * BN;

    const int x_blocks = (t + 15) >> 4;
    const __amdgpu_buffer_rsrc_t xr = w4_make_rsrc(xq + (size_t)(m0 >> 4) * kt * 1024, (unsigned)min(x_blocks - (m0 >> 4), BM / 16) * (unsigned)kt * 1024u);
    // first row block of the wave's columns and what is left of the matrix behind it
    const int wrb = (n0 >> 4) + wave * (GLU ? 2 : 4), w_end = GLU ? half_rb : row_blocks;
    auto w_rsrc = [&](int first, int count) {
        return w4_make_rsrc(wt + (size_t)(count > 0 ? first : 0) * kt * 1024, (unsigned)max(count, 0) * (unsigned)kt * 1024u);
    };
    const __amdgpu_buffer_rsrc_t wr0 = w_rsrc(wrb, min(w_end - wrb, GLU ? 2 : 4)),
                                 wr1 = GLU ? w_rsrc(half_rb + wrb, min(w_end - wrb, 2)) : wr0;
    typedef __attribute__((address_space(3))) char lds_char_t;
    lds_char_t* const lds_base = (lds_char_t*)lds;
    // stage in LDS: [row block][two k tiles] of 1 KiB
    unsigned xa[NA];
#pragma unroll
    for (int i = 0; i < NA; i++) {
        const int tile = i * 4 + wave;
        xa[i] = (unsigned)(tile >> 1) * (unsigned)kt * 1024u + (tile & 1) * 1024u + lane * 16u;
    }
    auto load_x = [&](int s, int buf) {
#pragma unroll
        for (int i = 0; i < NA; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void*)(lds_base + buf * STAGE + (i * 4 + wave) * 1024), 16,
                                                     xa[i], s * 2048, 0, 0);
    };
    unsigned wo[2];
#pragma unroll
    for (int ni = 0; ni < 2; ni++)
        wo[ni] = (unsigned)((GLU ? 0 : ni * 2) + (nl >> 4)) * (unsigned)kt * 1024u + kh * 256u + (nl & 15) * 16u;
    i4_t b[2][2][4];
    auto load_w = [&](i4_t (&d)[2][4], int s) {
#pragma unroll
        for (int ni = 0; ni < 2; ni++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                d[ni][q] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(ni ? wr1 : wr0, wo[ni] + q * 512, s * 2048, 0));
    };
    i16_t acc[MI][2];
#pragma unroll
    for (int mi = 0; mi < MI; mi++)
#pragma unroll
        for (int ni = 0; ni < 2; ni++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[mi][ni][e] = 0;
    const char* const frag = lds + ((nl >> 4) * 2048 + kh * 256 + (nl & 15) * 16);
    auto products = [&](const i4_t (&w)[2][4], int buf) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            i4_t a[MI];
#pragma unroll
            for (int mi = 0; mi < MI; mi++) a[mi] = *reinterpret_cast<const i4_t*>(frag + buf * STAGE + mi * 4096 + q * 512);
#pragma unroll
            for (int ni = 0; ni < 2; ni++)
#pragma unroll
                for (int mi = 0; mi < MI; mi++) acc[mi][ni] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[ni][q], a[mi], acc[mi][ni], 0, 0, 0);
        }
    };
    const int stages = kt >> 1;
    load_x(0, 0);
    load_w(b[0], 0);
    w4_dma_barrier();
    for (int s = 0; s < stages; s += 2) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (s + h < stages) {
                if (s + h + 1 < stages) {
                    load_x(s + h + 1, h ^ 1);  // the buffer that stage s + h - 1 was read from: every wave is past its barrier
                    load_w(b[h ^ 1], s + h + 1);
                }
                products(b[h], h);
                w4_dma_barrier();
            }
        }
    }
    // D register e of lane (nl, kh): output column 8 (e / 4) + 4 kh + e % 4, row nl
#pragma unroll
    for (int mi = 0; mi < MI; mi++) {
        const int m = m0 + mi * 32 + nl;
        if (m >= t) continue;
        const float sx = xs[m];
#pragma unroll
        for (int ni = 0; ni < (GLU ? 1 : 2); ni++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int c = n0 + wave * (GLU ? 32 : 64) + ni * 32 + g * 8 + kh * 4;
                if (c >= out_n) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[e] = (float)acc[mi][ni][g * 4 + e] * sx * ws[c + e];
                    if (GLU) v[e] = w4_act_mul(v[e], (float)acc[mi][1][g * 4 + e] * sx * ws[out_n + c + e], act);
                }
                w8_store4(y, (size_t)m * out_n + c, out_n - c, v, y_type);
            }
    }
}

#define W8_TILED(NAME, MI, GLU)                                                                                                   \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                           int kt, int t, int y_type, int act) {                                  \
        tiled_body<MI, GLU>(wt, ws, xq, xs, y, n, kt, t, y_type, act);                                                            \
    }
W8_TILED(w4a16_w8a8_tiled_m128, 4, false)
W8_TILED(w4a16_w8a8_tiled_m128_glu, 4, true)
