// Quantisation of activation rows to e4m3 with a scale for each block of 128 k.  The scale is a power of two, the least that brings the block's largest
// magnitude to 448 or below: every quotient is then exact and the conversion its only rounding (to nearest, halves to even), and since the numbers float, a
// step up to twice as large loses nothing but the last of 18 binary orders below the largest.
#include "f8_common.hpp"

// A thread per 16 columns, eight lanes to a block; a wave takes LR = 1, 4 or 8 neighbouring rows (tiles of R = 1, 4, 16 rows), whose 16-byte chunks lie side by
// side, and 8 / LR blocks of each.  Whole blocks are written: zeros behind the row's end, which meet zero weights as numbers.
template <int T>
__device__ __forceinline__ void f8_quant_body(const void* __restrict__ x, size_t ldx, int k, int kb, int R, char* __restrict__ q, float* __restrict__ s,
                                              int t, size_t s_ld) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = R == 16 ? 8 : R;
    const int group = blockIdx.x * (R == 16 ? 2 : 1) + (R == 16 ? wave & 1 : 0);  // of lr rows: a tile's two to neighbouring waves
    const int per = 8 / lr, ahead = R == 16 ? wave >> 1 : wave, stride = R == 16 ? 2 : 4;
    const int row = group * lr + (lane >> 3) % lr, b = ((int)blockIdx.y * stride + ahead) * per + (lane >> 3) / lr, c = b * 8 + (lane & 7);
    if (row >= t || b >= kb) return;  // whole runs of eight lanes
    const char* const xr = static_cast<const char*>(x) + (size_t)row * ldx * (T == Q8_F32 ? 4 : 2);
    F8Run<T> v;
    v.load(xr, c * 16, k - c * 16);
    float by;
    const float step = f8_step(f8_block_max(v.most(0)), by);
    const u4_t o = v.pack(by, !(step > 0.f));
    *reinterpret_cast<u4_t*>(q + q8_chunk_at(row, c, 2 * kb, R)) = o;
    if ((lane & 7) == 0) s[(size_t)b * s_ld + row] = step;
}

#define F8_QUANT(NAME, T)                                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void NAME(const void* x, size_t ldx, int k, int kb, int R, char* q, float* s, int t, size_t s_ld) { \
        f8_quant_body<T>(x, ldx, k, kb, R, q, s, t, s_ld);                                                                 \
    }
F8_QUANT(w4a16_quant_rows_f8_f32, Q8_F32)
F8_QUANT(w4a16_quant_rows_f8_f16, Q8_F16)
F8_QUANT(w4a16_quant_rows_f8_bf16, Q8_BF16)

// w4a16_norm_resid (glue.hip) and the quantisation of its f32 result in one pass: the same arithmetic in the same order, so the rows are those of the two
// launches bit for bit.  x <- x + ab; xn = x * inv * nw[w_off + c] is rounded twice and never stored.
// A row to a workgroup, four neighbours to a thread, whose four partial sums are those of four neighbouring threads of the 1024 there; 32 lanes have a block of 128.  What bounds few rows is
// the chain of one: loads, sum, stores; so no branch stands between its loads, which the compiler would wait behind.  5120 elements: 1 row 3.6 us, 300 8.0, 4096 53.5 (5.1 TB/s); one element to
// a thread of 1024: 4.2, 12.0 and 64.
template <int N>  // rounds of 1024 elements
__device__ __forceinline__ void f8_norm_body(float* __restrict__ x, const float* __restrict__ nw, const float* __restrict__ ab, char* __restrict__ q, float* __restrict__ s,
                                             int w_off, int hidden, int kb, int R, int row, size_t s_ld, float* red) {
    const int tid = threadIdx.x;
    float* const xr = x + (size_t)row * hidden;
    const float* const ar = ab + (size_t)row * hidden;
    // Buffers of one row: elements behind its end read as 0 and are not written.  All loads ahead of the first use, with no branch between them.
    const __amdgpu_buffer_rsrc_t xb = w4_make_rsrc(xr, (unsigned)hidden * 4u), ab_r = w4_make_rsrc(ar, (unsigned)hidden * 4u), wb = w4_make_rsrc(nw + w_off, (unsigned)hidden * 4u);
    f4_t v[N], y[N], more[N], ss = {0.f, 0.f, 0.f, 0.f};
    const int at = tid * 16;
    if (hidden % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            v[j] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(xb, at + j * 4096, 0, 0));
            more[j] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(ab_r, at + j * 4096, 0, 0));
            y[j] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(wb, at + j * 4096, 0, 0));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[j][e] = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(xb, at + j * 4096 + e * 4, 0, 0));
                more[j][e] = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(ab_r, at + j * 4096 + e * 4, 0, 0));
                y[j][e] = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(wb, at + j * 4096 + e * 4, 0, 0));
            }
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        v[j] = v[j] + more[j];
#pragma unroll
        for (int e = 0; e < 4; e++) ss[e] = __builtin_fmaf(v[j][e], v[j][e], ss[e]);
    }
    *reinterpret_cast<f4_t*>(red + tid * 4) = ss;
    __syncthreads();
    const float inv = 1.0f / sqrtf(q8_norm_total(red) / (float)hidden + 1e-6f);
    unsigned most[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        most[j] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float p = v[j][e] * inv;
            asm volatile("" : "+v"(p));  // two roundings, never one fused product
            y[j][e] = j * 1024 + tid * 4 + e < hidden ? p * y[j][e] : 0.f;
            most[j] = max(most[j], q8_mag(y[j][e]));
        }
        most[j] = f8_half_wave_max(most[j]);
    }
    if (hidden % 4 == 0) {
#pragma unroll
        for (int j = 0; j < N; j++) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v[j]), xb, at + j * 4096, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)v[j][e]), xb, at + j * 4096 + e * 4, 0, 0);
    }
    // Whole blocks: behind the row's end the bytes are 0.  A buffer of the row's tiles: blocks that are not there are not written.
    const __amdgpu_buffer_rsrc_t qb = w4_make_rsrc(q + (size_t)(row / R) * R * kb * 128, (unsigned)R * (unsigned)kb * 128u);
    float step[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        float by;
        step[j] = f8_step(most[j], by);
        const unsigned four = f8_pack4(y[j][0], y[j][1], y[j][2], y[j][3], by, !(step[j] > 0.f));
        __builtin_amdgcn_raw_buffer_store_b32(four, qb, ((j * 64 + (tid >> 2)) * R + row % R) * 16 + (tid & 3) * 4, 0, 0);
    }
    if ((tid & 31) == 0) {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j * 8 + (tid >> 5) < kb) s[(size_t)(j * 8 + (tid >> 5)) * s_ld + row] = step[j];
    }
}

#define F8_NORM_THREADS 256
extern "C" __global__ __launch_bounds__(F8_NORM_THREADS) void w4a16_norm_resid_f8(float* __restrict__ x, const float* __restrict__ nw,
                                                                                  const float* __restrict__ ab, char* __restrict__ q,
                                                                                  float* __restrict__ s, int w_off, int hidden, int kb, int R, int t, size_t s_ld) {
    __shared__ __attribute__((aligned(16))) float red[1024];
    const int row = q8_row_of_block(R);
    if (row >= t) return;
    if (hidden <= 2048) f8_norm_body<2>(x, nw, ab, q, s, w_off, hidden, kb, R, row, s_ld, red);
    else if (hidden <= 5120) f8_norm_body<5>(x, nw, ab, q, s, w_off, hidden, kb, R, row, s_ld, red);
    else f8_norm_body<8>(x, nw, ab, q, s, w_off, hidden, kb, R, row, s_ld, red);
}
