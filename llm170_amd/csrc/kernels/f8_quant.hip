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
// launches bit for bit.  x <- x + ab; xn = x * inv * nw[w_off + c] is rounded twice and never stored.  A block of 128 columns is two waves' of one round.
extern "C" __global__ __launch_bounds__(1024) void w4a16_norm_resid_f8(float* __restrict__ x, const float* __restrict__ nw,
                                                                       const float* __restrict__ ab, char* __restrict__ q,
                                                                       float* __restrict__ s, int w_off, int hidden, int kb, int R, int t, size_t s_ld) {
    __shared__ float red[1024];
    __shared__ unsigned redm[8][16];
    __shared__ __attribute__((aligned(16))) char line[8192];
    const int tid = threadIdx.x, wave = tid >> 6, row = q8_row_of_block(R);
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
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = j * 1024 + tid;
        float p = v[j] * inv;
        asm volatile("" : "+v"(p));  // two roundings, never one fused product
        y[j] = p * y[j];
        if (c < hidden) x[base + c] = v[j];
        if (j * 1024 < hidden) {  // uniform
            const unsigned m = q8_wave_max(c < hidden ? q8_mag(y[j]) : 0u);
            if ((tid & 63) == 0) redm[j][wave] = m;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (j * 1024 >= hidden) continue;
        const int c = j * 1024 + tid;
        float by;
        const float step = f8_step(max(redm[j][wave & ~1], redm[j][wave | 1]), by);
        line[c] = (char)f8_pack4(c < hidden ? y[j] : 0.f, 0.f, 0.f, 0.f, by, !(step > 0.f));
        if ((tid & 127) == 0 && c < hidden) s[(size_t)(c >> 7) * s_ld + row] = step;
    }
    __syncthreads();
    // whole blocks: behind the row's end the bytes are 0
    if (tid < kb * 8) *reinterpret_cast<u4_t*>(q + q8_chunk_at(row, tid, 2 * kb, R)) = *reinterpret_cast<const u4_t*>(line + tid * 16);
}
