// Quantisation of activation rows to int8 with one scale per row, and the re-layout of int8 weights at upload.
#include "q8_common.hpp"

// Largest of one value per thread over the workgroup.
__device__ __forceinline__ unsigned quant_block_max(unsigned m, unsigned* red, int waves) {
#pragma unroll
    for (int st = 32; st > 0; st >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, st));
    if (waves == 1) return m;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < waves; w++) m = max(m, red[w]);
    return m;
}

// s[r] = step of row r, q = round(x / s) in tiles of R rows.  A workgroup per row, a thread per 16 columns and round; the first
// KEEP rounds stay in registers between the two passes over the row, what lies behind them is read again from the cache.
#define QUANT_KEEP 2
template <int T>
__device__ __forceinline__ void quant_body(const void* __restrict__ x, size_t ldx, int k, int kt, int R, char* __restrict__ q,
                                           float* __restrict__ s, int t, int threads) {
    __shared__ unsigned red[16];
    // Sixteen neighbouring rows share their 256-byte runs of the tiles: they go to one XCD (block b runs on XCD b % 8), whose
    // L2 joins their 16-byte pieces.
    const int b = blockIdx.x, row = R == 16 ? ((b >> 7) * 8 + (b & 7)) * 16 + ((b >> 3) & 15) : b;
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
        u4_t o;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            unsigned b4 = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) b4 |= ((unsigned)q8_round(w[4 * j + e], step, r) & 0xffu) << (8 * e);
            o[j] = b4;
        }
        *reinterpret_cast<u4_t*>(q + q8_chunk_at(row, c, kt, R)) = o;
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

// w4a16_norm_resid (glue.hip) and the quantisation of its f32 result in one pass: the same arithmetic in the same order, so the
// rows are those of the two launches bit for bit.  x <- x + ab; xn = x * inv * nw[w_off + c] is rounded twice and never stored.
extern "C" __global__ __launch_bounds__(1024) void w4a16_norm_resid_q8(float* __restrict__ x, const float* __restrict__ nw,
                                                                       const float* __restrict__ ab, char* __restrict__ q,
                                                                       float* __restrict__ s, int w_off, int hidden, int kt, int R) {
    __shared__ float red[1024];
    __shared__ unsigned redm[16];
    const int tid = threadIdx.x, row = blockIdx.x;
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
    red[tid] = ss;
    __syncthreads();
    for (int st = 512; st >= 64; st >>= 1) {
        if (tid < st) red[tid] = red[tid] + red[tid + st];
        __syncthreads();
    }
    float r = red[tid & 63];
#pragma unroll
    for (int st = 32; st > 0; st >>= 1) r = r + __shfl_down(r, st);
    r = __shfl(r, 0);
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
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = j * 1024 + tid;
        if (c < hidden) q[q8_chunk_at(row, c >> 4, kt, R) + (c & 15)] = (char)q8_round(y[j], step, rs);
    }
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
