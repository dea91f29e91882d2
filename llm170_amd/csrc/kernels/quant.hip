// Quantisation of activation rows to int8 with one scale per row, and the re-layout of int8 weights at upload.
#include "q8_common.hpp"

// Largest of one value per thread over the workgroup.
__device__ __forceinline__ unsigned quant_block_max(unsigned m, unsigned* red, int waves) {
    m = q8_wave_max(m);
    if (waves == 1) return m;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < waves; w++) m = max(m, red[w]);
    return m;
}

// s[r] = step of row r, q = round(x / s) in tiles of R rows.  A workgroup per row, a thread per 16 columns and round; the first
// KEEP rounds stay in registers between the two passes over the row, what lies behind them is read again from the cache.
// Launches back to back: 4096 x 5120 f16 19.0 us, 300 x 17408 8.7, 4096 x 17408 51.6.  The waves wait (65 % of their cycles at 4096 x 5120; for the
// issue of instructions 10 %): a workgroup loads its row, reduces it and stores it one after another.
#define QUANT_KEEP 2
template <int T>
__device__ __forceinline__ void quant_body(const void* __restrict__ x, size_t ldx, int k, int kt, int R, char* __restrict__ q,
                                           float* __restrict__ s, int t, int threads) {
    __shared__ unsigned red[16];
    const int row = q8_row_of_block(R);
    if (row >= t) return;
    const char* const xr = static_cast<const char*>(x) + (size_t)row * ldx * (T == Q8_F32 ? 4 : 2);
    const int chunks = (k + 15) >> 4;
    float v[QUANT_KEEP][16];
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < QUANT_KEEP; i++) {
        const int c = threadIdx.x + i * threads;
        q8_load16<T>(xr, (size_t)c * 16, k - c * 16, v[i]);
    }
#pragma unroll
    for (int i = 0; i < QUANT_KEEP; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) m = max(m, q8_mag(v[i][e]));
    for (int c = threadIdx.x + QUANT_KEEP * threads; c < chunks; c += threads) {
        float w[16];
        q8_load16<T>(xr, (size_t)c * 16, k - c * 16, w);
#pragma unroll
        for (int e = 0; e < 16; e++) m = max(m, q8_mag(w[e]));
    }
    const float step = q8_step(quant_block_max(m, red, threads >> 6)), r = q8_recip(step);
    if (threadIdx.x == 0) s[row] = step;
    auto put = [&](int c, const float (&w)[16]) {
        unsigned o[4];
        q8_pack<16>(w, step, r, o);
        *reinterpret_cast<u4_t*>(q + q8_chunk_at(row, c, kt, R)) = (u4_t){o[0], o[1], o[2], o[3]};
    };
#pragma unroll
    for (int i = 0; i < QUANT_KEEP; i++) {
        const int c = threadIdx.x + i * threads;
        if (c < chunks) put(c, v[i]);
    }
    for (int c = threadIdx.x + QUANT_KEEP * threads; c < chunks; c += threads) {
        float w[16];
        q8_load16<T>(xr, (size_t)c * 16, k - c * 16, w);
        put(c, w);
    }
}

#define QUANT_KERNEL(NAME, T)                                                                                              \
    extern "C" __global__ __launch_bounds__(1024) void NAME(const void* x, size_t ldx, int k, int kt, int R, char* q, float* s, int t, int threads) { \
        quant_body<T>(x, ldx, k, kt, R, q, s, t, threads);                                                                          \
    }
QUANT_KERNEL(w4a16_quant_rows_f32, Q8_F32)
QUANT_KERNEL(w4a16_quant_rows_f16, Q8_F16)
QUANT_KERNEL(w4a16_quant_rows_bf16, Q8_BF16)

// Few rows: their number cannot hide the way to a row's maximum and back.  A row has up to sixteen waves, four columns per thread and
// round, the first FEW_KEEP rounds in registers; and where it has several rounds, as many workgroups (gridDim.y), each of which looks for the
// maximum of the whole row and quantises its own round.
#define QUANT_FEW_KEEP 5
template <int T>
__device__ __forceinline__ void few_load(const char* row, int c, int k, float (&v)[4]) {
    if (c + 4 <= k) {
        if (T == Q8_F32) {
            const u4_any_t w = *reinterpret_cast<const u4_any_t*>(row + (size_t)c * 4);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = q8_f32(w[e]);
        } else {
            const u2_any_t w = *reinterpret_cast<const u2_any_t*>(row + (size_t)c * 2);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                v[2 * e] = T == Q8_F16 ? q8_half(w[e], 0) : q8_bf16(w[e] & 0xffffu);
                v[2 * e + 1] = T == Q8_F16 ? q8_half(w[e], 1) : q8_f32(w[e] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = c + e < k ? q8_load1<T>(row, (size_t)(c + e)) : 0.f;
    }
}

template <int T>
__device__ __forceinline__ void few_body(const void* __restrict__ x, size_t ldx, int k, int kt, int R, char* __restrict__ q, float* __restrict__ s,
                                         int threads) {
    __shared__ unsigned red[16];
    const int row = blockIdx.x, step_c = threads * 4;
    const char* const xr = static_cast<const char*>(x) + (size_t)row * ldx * (T == Q8_F32 ? 4 : 2);
    const int c0 = threadIdx.x * 4;
    float v[QUANT_FEW_KEEP][4];
#pragma unroll
    for (int i = 0; i < QUANT_FEW_KEEP; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[i][e] = 0.f;
        if (i * step_c < k) few_load<T>(xr, c0 + i * step_c, k, v[i]);  // uniform
    }
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < QUANT_FEW_KEEP; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) m = max(m, q8_mag(v[i][e]));
#pragma unroll 1
    for (int c = c0 + QUANT_FEW_KEEP * step_c; c < k; c += step_c) {
        float w[4];
        few_load<T>(xr, c, k, w);
#pragma unroll
        for (int e = 0; e < 4; e++) m = max(m, q8_mag(w[e]));
    }
    const float step = q8_step(quant_block_max(m, red, threads >> 6)), r = q8_recip(step);
    const int part = blockIdx.y, c = c0 + part * step_c;
    if (threadIdx.x == 0 && part == 0) s[row] = step;
    if (c >= ((k + 15) & ~15)) return;  // whole chunks of 16 are written, with zeros behind the row's end
    float w[4];
    if (part < QUANT_FEW_KEEP) {
#pragma unroll
        for (int i = 0; i < QUANT_FEW_KEEP; i++)
            if (i == part)
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = v[i][e];
    } else {
        few_load<T>(xr, c, k, w);
    }
    unsigned o[1];
    q8_pack<4>(w, step, r, o);
    *reinterpret_cast<unsigned*>(q + q8_chunk_at(row, c >> 4, kt, R) + (c & 15)) = o[0];
}

#define QUANT_FEW(NAME, T)                                                                                                 \
    extern "C" __global__ __launch_bounds__(1024) void NAME(const void* x, size_t ldx, int k, int kt, int R, char* q, float* s, int, int threads) { \
        few_body<T>(x, ldx, k, kt, R, q, s, threads);                                                                      \
    }
QUANT_FEW(w4a16_quant_few_f32, Q8_F32)
QUANT_FEW(w4a16_quant_few_f16, Q8_F16)
QUANT_FEW(w4a16_quant_few_bf16, Q8_BF16)

// w4a16_norm_resid (glue.hip) and the quantisation of its f32 result in one pass: the same arithmetic in the same order, so the
// rows are those of the two launches bit for bit.  x <- x + ab; xn = x * inv * nw[w_off + c] is rounded twice and never stored.
// Launches back to back, cold rows: 4096 x 5120 64 us (w4a16_norm_resid, which writes f32, 75; the bytes at a copy's rate 53), 300 x 5120 9.6 (9.0).  On the
// same rows again and again 50 and 7.2; with byte stores and rows of a tile on all XCDs 59 and 8.7.
extern "C" __global__ __launch_bounds__(1024) void w4a16_norm_resid_q8(float* __restrict__ x, const float* __restrict__ nw,
                                                                       const float* __restrict__ ab, char* __restrict__ q,
                                                                       float* __restrict__ s, int w_off, int hidden, int kt, int R, int t) {
    __shared__ float red[1024];
    __shared__ unsigned redm[16];
    __shared__ __attribute__((aligned(16))) char line[8192];
    const int tid = threadIdx.x, row = q8_row_of_block(R);
    if (row >= t) return;
    const size_t base = (size_t)row * hidden;
    float v[8], y[8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = j * 1024 + tid;
        v[j] = 0.0f;
        y[j] = 0.0f;
        if (c < hidden) {
            v[j] = x[base + c] + ab[base + c];
            y[j] = nw[w_off + c];
            ss = __builtin_fmaf(v[j], v[j], ss);
        }
    }
    const float r = q8_norm_sum(ss, red);
    const float inv = 1.0f / sqrtf(r / (float)hidden + 1e-6f);
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = j * 1024 + tid;
        float p = v[j] * inv;
        asm volatile("" : "+v"(p));  // two roundings, never one fused product
        y[j] = p * y[j];
        if (c < hidden) {
            m = max(m, q8_mag(y[j]));
            x[base + c] = v[j];
        }
    }
    const float step = q8_step(quant_block_max(m, redm, 16)), rs = q8_recip(step);
    if (tid == 0) s[row] = step;
    unsigned o[2];
    q8_pack<8>(y, step, rs, o);
#pragma unroll
    for (int j = 0; j < 8; j++) line[j * 1024 + tid] = (char)(o[j / 4] >> (8 * (j % 4)));
    __syncthreads();
    // whole chunks: behind the row's end v and y, and so the bytes, are 0
    if (tid * 16 < hidden) *reinterpret_cast<u4_t*>(q + q8_chunk_at(row, tid, kt, R)) = *reinterpret_cast<const u4_t*>(line + tid * 16);
}

// Weights int8 [n][k] -> tiles [row_blocks][kt], zeros behind n and k: a thread per 16-byte chunk of the result.
extern "C" __global__ __launch_bounds__(256) void w4a16_tile_w8(const signed char* __restrict__ w, u4_t* __restrict__ out, size_t n, int k,
                                                                int kt, size_t chunks) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (size_t)gridDim.x * 256) {
        const size_t tile = i >> 6, row = tile / kt * 16 + (i & 15);
        const int col = (int)(tile % kt) * 64 + (int)((i >> 4) & 3) * 16;
        u4_t o = {0, 0, 0, 0};
        if (row < n && col < k) {
            const signed char* const p = w + row * (size_t)k + col;
            const int left = min(16, k - col);
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (e < left) o[e >> 2] |= ((unsigned)p[e] & 0xffu) << (8 * (e & 3));
        }
        out[i] = o;
    }
}
