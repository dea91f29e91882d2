// FP8 linears:  y[m][n] = sum_b sx[b][m] * sw[n / 128][b] * sum_{k in b} q[m][k] w[n][k],  q and w e4m3 in tiles (q8_common.hpp, two k tiles
// to a block of 128), an f32 scale for each 128 k of a row and for each 128 x 128 of the weights.  A block's products are summed from zero on the matrix
// units and enter the running sum with one fused multiply-add.  Gated form: rows 0..n/2 of w are a gate, the rest its values, y[m][c] = act(gate) * value.
//
// Which product.  The e4m3 matrix instruction aligns products to the largest of their group and drops what lies 2^-14 and more below it: on normal
// numbers 1.6e-5 of the results' size, 4.2 PFLOP/s alone (16x16x128; 32x32x64 3.8), 3.5 with the scaling.  As f16, which holds every e4m3 number, the same
// sums are those of 32 bits (1e-8), at the f16 instruction's 1.6.  So f16 for f32 results, up to 64 rows, where
// the weight stream is what takes the time, and for gated results of up to 1024 rows: the next linear quantises those, and a number that falls to the other side of one of its
// roundings shows 4000 times what was dropped (two linears at 300 rows: 1.4e-3 of their result's size, with f16 products 2e-4 to 5e-4).  e4m3 for the other 16-bit results, whose own rounding
// is ten times as large and more: 5120 x 17408 at 300 rows 53.5 us, with f16 products 70.8.
#include "f8_common.hpp"

typedef int i8_t __attribute__((ext_vector_type(8)));

// Two of four e4m3 numbers as f16, and eight, exactly
__device__ __forceinline__ unsigned f8_to_f16_pair(unsigned four, bool high) {
    return __builtin_bit_cast(unsigned, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)four, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)four, 1.0f, false));
}
__device__ __forceinline__ h8_t f8_to_f16(unsigned lo, unsigned hi) {
    const h2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
    const h2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
    return (h8_t){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float f8_lane(float v, int lane) { return q8_f32((unsigned)__builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }

// ------------------------------------------------------------------------------------------------ up to 64 rows
// As the int8 kernel for few rows (w8a8.hip): a workgroup's waves take consecutive runs of a k slice of the same RB row blocks (16 outputs each), weights as whole
// tiles straight in registers, DEPTH blocks of them in flight, TT tiles of 16 activation rows from the L2.  The waves' sums are added in the order of
// the waves in LDS and the k slices' in their order by the last workgroup: the same bits every time.  The weights' scales of a run lie one to a lane.
//
// Few rows of floats (XT: their type) are quantised on the way: a workgroup's threads take the blocks of its k slice, 16 elements of a row each, once, and leave
// them in LDS, 132 bytes with its scale, while the first weights are on their way: up to F8_FLOAT_BLOCKS of them, more take longer than a launch that does it.
#define F8_FLOAT_BLOCKS 128
template <int RB, int TT, bool GLU, int XT>
__device__ __forceinline__ void f8_skinny_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                               const float* __restrict__ xs, size_t ldx, int k_in, void* __restrict__ y, int n, int kb, int t, int R, int y_type,
                                               int act, int W, int nks, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr bool FLOATS = XT != F8_ROWS;
    static_assert(!FLOATS || TT == 1, "floats: up to 16 rows");
    constexpr int TILES = RB * TT, DEPTH = TILES == 1 ? 4 : TILES <= 8 && TT < 4 ? 2 : 1, SLOTS = TILES <= 4 ? 8 : 4, XD = FLOATS ? 1 : DEPTH;
    __shared__ float sums[SLOTS][TILES][4][64];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_blocks = (n + 15) >> 4, half_rb = GLU ? row_blocks >> 1 : 0;
    // row block of slot i: gated, slots 2j and 2j + 1 are a gate's and its values'
    auto block_of = [&](int i) { return GLU ? blockIdx.x * (RB / 2) + i / 2 + (i & 1 ? half_rb : 0) : blockIdx.x * RB + i; };
    const int last = (GLU ? half_rb : row_blocks) - 1;
    const int tok = lane & 15, kg = lane >> 4;
    const int ks = blockIdx.y % (unsigned)nks, group = blockIdx.y / (unsigned)nks, groups = gridDim.y / (unsigned)nks;
    const int runs = nks * W, run = ks * W + wave;
    const int m0 = group * TT * 16, x_last = (t - 1) >> 4;  // rows of the group, and the last tile of 16 that there is
    const int lo = (int)((long long)kb * run / runs), hi = (int)((long long)kb * (run + 1) / runs);
    // floats: this thread's first runs of 16 elements, asked for ahead of the weights, whose loads they would otherwise wait for; chunk i & 7 of row and block i >> 3
    extern __shared__ __attribute__((aligned(16))) char lds_x[];  // [block of the slice][chunk][row] of 16 bytes, then [block][row] scales
    constexpr int PRE = XT == Q8_F32 ? 2 : 4;
    constexpr int RUN = FLOATS ? XT : Q8_F16;  // a type that there is
    const int s_lo = (int)((long long)kb * ks / nks), items = FLOATS ? ((int)((long long)kb * (ks + 1) / nks) - s_lo) * t * 8 : 0;
    F8Run<RUN> pre[PRE];
    auto load_run = [&](F8Run<RUN>& v, int i) {
        const int br = i >> 3, block = br / t, c = (s_lo + block) * 8 + (i & 7);
        v.load(xq + (size_t)(br - block * t) * ldx * (RUN == Q8_F32 ? 4 : 2), c * 16, k_in - c * 16);
    };
    auto put_run = [&](const F8Run<RUN>& v, int i) {
        const int br = i >> 3, block = br / t;
        float by;
        const float step = f8_step(f8_block_max(v.most(0)), by);
        *reinterpret_cast<u4_t*>(lds_x + ((size_t)(block * 8 + (i & 7)) * t + (br - block * t)) * 16) = v.pack(by, !(step > 0.f));
        if ((i & 7) == 0) *reinterpret_cast<float*>(lds_x + (size_t)items * 16 + br * 4) = step;
    };
    if constexpr (FLOATS) {
#pragma unroll
        for (int i = 0; i < PRE; i++)
            if ((int)threadIdx.x + i * W * 64 < items) load_run(pre[i], threadIdx.x + i * W * 64);
    }
    const char* wp[RB];
    const float* wsp[RB];
    float wsv[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) {
        int b = block_of(i);
        if (GLU) b = min(b - (i & 1 ? half_rb : 0), last) + (i & 1 ? half_rb : 0);  // slots past the end read the last block, not stored
        else b = min(b, last);
        wp[i] = wt + (size_t)b * kb * 2048 + lane * 16;
        wsp[i] = ws + (size_t)(b >> 3) * kb;
        wsv[i] = wsp[i][min(lo + lane, kb - 1)];
    }
    // activations: tiles of R rows, [k tile][kg][R] chunks
    const char* const xp = xq + ((size_t)kg * R + tok % R) * 16;
    const size_t x_tile = (size_t)R * 64, x_block = x_tile * 2 * kb;
    const int lds_at = (kg * t + tok % t) * 16, lds_tile = t * 64;  // floats: the lane's chunk of the slice's first block
    f4_t acc[RB][TT];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = (f4_t){0.f, 0.f, 0.f, 0.f};
    u4_t wv[DEPTH][RB][2], xv[XD][TT][2];
    float xsv[XD][TT];
    auto load_w = [&](int d, int i, int k) {
        // Non-temporal weights: 34816 x 5120 gated int8 at t = 1 31.3 us, else 35.2
#pragma unroll
        for (int h = 0; h < 2; h++) wv[d][i][h] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(wp[i] + (size_t)k * 2048 + h * 1024));
    };
    auto load_x = [&](int d, int k) {
        if constexpr (FLOATS) {
            const char* const p = lds_x + lds_at + (2 * (k - s_lo)) * lds_tile;
            xv[d][0][0] = *reinterpret_cast<const u4_t*>(p);
            xv[d][0][1] = *reinterpret_cast<const u4_t*>(p + lds_tile);
            xsv[d][0] = *reinterpret_cast<const float*>(lds_x + (size_t)items * 16 + ((k - s_lo) * t + tok % t) * 4);
        } else {
#pragma unroll
            for (int j = 0; j < TT; j++) {
#pragma unroll
                for (int h = 0; h < 2; h++) xv[d][j][h] = *reinterpret_cast<const u4_t*>(xp + min((m0 >> 4) + j, x_last) * x_block + (2 * k + h) * x_tile);
                xsv[d][j] = xs[(size_t)k * t + min(m0 + j * 16 + tok, t - 1)];
            }
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
        if (lo + d >= hi) continue;
#pragma unroll
        for (int i = 0; i < RB; i++) load_w(d, i, lo + d);
        if (!FLOATS) load_x(d, lo + d);
    }
    if constexpr (FLOATS) {
#pragma unroll
        for (int i = 0; i < PRE; i++)
            if ((int)threadIdx.x + i * W * 64 < items) put_run(pre[i], threadIdx.x + i * W * 64);
        for (int i = threadIdx.x + PRE * W * 64; i < items; i += W * 64) {
            F8Run<RUN> v;
            load_run(v, i);
            put_run(v, i);
        }
        w8_lds_done();
        w8_lds_barrier();
        if (lo < hi) load_x(0, lo);
    }
    int base = lo;  // of the 64 blocks whose scales are in the lanes
    for (int k = lo; k < hi; k += DEPTH) {
        if (k + DEPTH > base + 64) {
            base = k;
#pragma unroll
            for (int i = 0; i < RB; i++) wsv[i] = wsp[i][min(base + lane, kb - 1)];
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            if (k + d < hi) {
                const int next = k + d + DEPTH;
                h8_t x[TT][4];
                float sx[TT];
                constexpr int AT = FLOATS ? 0 : 1;
#pragma unroll
                for (int j = 0; j < TT; j++) {
                    sx[j] = xsv[d * AT][j];
#pragma unroll
                    for (int c = 0; c < 4; c++) x[j][c] = f8_to_f16(xv[d * AT][j][c / 2][c % 2 * 2], xv[d * AT][j][c / 2][c % 2 * 2 + 1]);
                }
                if (FLOATS ? k + d + 1 < hi : next < hi) load_x(d * AT, FLOATS ? k + d + 1 : next);
#pragma unroll
                for (int i = 0; i < RB; i++) {
                    const float sw = f8_lane(wsv[i], k + d - base);
                    h8_t w[4];
                    f4_t p[TT];
#pragma unroll
                    for (int c = 0; c < 4; c++) w[c] = f8_to_f16(wv[d][i][c / 2][c % 2 * 2], wv[d][i][c / 2][c % 2 * 2 + 1]);
                    if (next < hi) load_w(d, i, next);
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int j = 0; j < TT; j++)
                            p[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[c], x[j][c], c == 0 ? (f4_t){0.f, 0.f, 0.f, 0.f} : p[j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < TT; j++) {
                        const float s = sx[j] * sw;
                        acc[i][j] = w4_fma4(p[j], (f4_t){s, s, s, s}, acc[i][j]);
                    }
                }
            }
        }
    }
    // The waves' sums: where there is a slot for each, all there; else the upper half's are added to the lower half's first
    int adders = W;
    auto put = [&](int slot) {
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < TT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) sums[slot][i * TT + j][e][lane] = acc[i][j][e];
    };
    if (SLOTS < 8 && W > SLOTS) {
        adders = (W + 1) >> 1;
        if (wave >= adders) put(wave - adders);
        __syncthreads();
        if (wave + adders < W) {
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int j = 0; j < TT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] += sums[wave][i * TT + j][e][lane];
        }
        __syncthreads();
    }
    if (wave < adders) put(wave);
    __syncthreads();
    // A wave finishes every W-th tile (gated: a gate and its values)
    auto total = [&](int tile) {
        f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < SLOTS; w++) {  // read at once; slots that were not written are left out
            f4_t o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = sums[w][tile][e][lane];
            v = w < adders ? v + o : v;
        }
        return v;
    };
    constexpr int U = GLU ? RB / 2 : RB;
    const unsigned own = group * gridDim.x + blockIdx.x;
    const size_t slice = (size_t)gridDim.x * groups * (TILES * 128);  // pairs of sums per k slice
    w8_pair_t* const mine = part + (size_t)own * (TILES * 128) + lane;
    if (nks > 1) {
        // Device-scope stores, complete before the ticket is drawn; device-scope loads behind the barrier that follows the ticket's return.
        // Neither is served from a cache that is not coherent.
#pragma unroll
        for (int u = 0; u < TILES; u++) {
            if (u % W != wave || m0 + (u % TT) * 16 + tok >= t) continue;
            const u4_t v = __builtin_bit_cast(u4_t, total(u));
            w8_pair_t* const p = mine + ks * slice + u * 128;
            __hip_atomic_store(p, (w8_pair_t)v[1] << 32 | v[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(p + 64, (w8_pair_t)v[3] << 32 | v[2], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) last_one = __hip_atomic_fetch_add(tickets + own, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nks - 1;
        __syncthreads();
        if (!last_one) return;
        if (threadIdx.x == 0) __hip_atomic_store(tickets + own, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    }
#pragma unroll
    for (int u = 0; u < U * TT; u++) {
        if (u % W != wave) continue;  // uniform for the wave
        const int i = GLU ? u / TT * 2 : u / TT, j = u % TT;
        const int b = block_of(i), m = m0 + j * 16 + tok, c = b * 16 + kg * 4;
        if (b > last || m >= t) continue;
        auto sum_of = [&](int i_) {
            if (nks == 1) return total(i_ * TT + j);
            f4_t v = {0.f, 0.f, 0.f, 0.f};
            const w8_pair_t* p = mine + (i_ * TT + j) * 128;
#pragma unroll 4
            for (int s = 0; s < nks; s++, p += slice) {
                const w8_pair_t a = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const w8_pair_t d = __hip_atomic_load(p + 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                v += (f4_t){q8_f32((unsigned)a), q8_f32((unsigned)(a >> 32)), q8_f32((unsigned)d), q8_f32((unsigned)(d >> 32))};
            }
            return v;
        };
        const f4_t sum = sum_of(i), sum_up = GLU ? sum_of(i + 1) : sum;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = GLU ? w4_act_mul(sum[e], sum_up[e], act) : sum[e];
        const int out_n = GLU ? n >> 1 : n;
        w8_store4(y, (size_t)m * out_n + c, out_n - c, v, y_type);
    }
}

#define F8_SKINNY(NAME, RB, TT, GLU)                                                                                              \
    extern "C" __global__ __launch_bounds__(512) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                           int kb, int t, int R, int y_type, int act, int waves, int nks, w8_pair_t* part,    \
                                                           int* tickets) {                                                        \
        f8_skinny_body<RB, TT, GLU, F8_ROWS>(wt, ws, xq, xs, 0, 0, y, n, kb, t, R, y_type, act, waves, nks, part, tickets);       \
    }
#define F8_SKINNY_X(NAME, RB, GLU, XT)                                                                                            \
    extern "C" __global__ __launch_bounds__(512) void NAME(const char* wt, const float* ws, const char* x, size_t ldx, int k, void* y, int n, \
                                                           int kb, int t, int y_type, int act, int waves, int nks, w8_pair_t* part,          \
                                                           int* tickets) {                                                        \
        f8_skinny_body<RB, 1, GLU, XT>(wt, ws, x, nullptr, ldx, k, y, n, kb, t, 16, y_type, act, waves, nks, part, tickets);      \
    }
#define F8_SKINNY_T(NAME, RB, GLU, SUFFIX)                           \
    F8_SKINNY(NAME##_t1##SUFFIX, RB, 1, GLU)                         \
    F8_SKINNY(NAME##_t2##SUFFIX, RB, 2, GLU)                         \
    F8_SKINNY(NAME##_t3##SUFFIX, RB, 3, GLU)                         \
    F8_SKINNY(NAME##_t4##SUFFIX, RB, 4, GLU)                         \
    F8_SKINNY_X(NAME##_f32##SUFFIX, RB, GLU, Q8_F32)                 \
    F8_SKINNY_X(NAME##_f16##SUFFIX, RB, GLU, Q8_F16)                 \
    F8_SKINNY_X(NAME##_bf16##SUFFIX, RB, GLU, Q8_BF16)
F8_SKINNY_T(w4a16_f8_skinny_r1, 1, false, )
F8_SKINNY_T(w4a16_f8_skinny_r2, 2, false, )
F8_SKINNY_T(w4a16_f8_skinny_r2, 2, true, _glu)
F8_SKINNY(w4a16_f8_skinny_r4_t2, 4, 2, false)
F8_SKINNY(w4a16_f8_skinny_r4_t3, 4, 3, false)
F8_SKINNY(w4a16_f8_skinny_r4_t2_glu, 4, 2, true)
F8_SKINNY(w4a16_f8_skinny_r4_t3_glu, 4, 3, true)

// ------------------------------------------------------------------------------------------------ tiles, any number of rows
// A workgroup of four waves has a tile of BM rows x 64 NB columns, each wave all of the rows and 16 NB of the columns.  Weights go straight into registers, each once; activations
// through registers into LDS, where the waves share them, with the products of their scales and the weights'.
// nks > 1: slices of k go to several workgroups, which hand their sums over as those of the kernels above do, added in the order of the slices.
//
// What bounds them, 34816 x 5120 gated (the instruction's rate alone: e4m3 4.2 PFLOP/s, f16 1.64):
//   128 x 256, e4m3: 650 us at 4096 rows, 2.23 PFLOP/s (64 x 128: 909); 5120 x 17408 350, 2.08; two waves a SIMD, 252 registers: the sums alone are 128
//   64 x 256, f16:   1214 us at 4096 rows, 1.20 PFLOP/s (64 x 128: 1341, LDS reads: four waves read each activation); 343 at 1000 rows, 124 at 300 (from HBM: 178 MB, 35 us)
// The end of a tile: slices of k are handed over and added in their order by the last workgroup, results stored
template <int J, int NB, bool GLU>
__device__ __forceinline__ void f8_finish(f4_t (&acc)[J][NB], int* last_one, int wrb, int m0, int out_n, int t, void* __restrict__ y, int y_type, int act, int nks, unsigned slice,
                                          unsigned tile, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int WAVES = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tok = lane & 15, kg = lane >> 4;
    if (nks > 1) {
        // [tile][slice][wave][block of 16 x 16][64 lanes] of 16 bytes, at device scope: past this XCD's L2
        constexpr int DEVICE = 16;  // sc1
        constexpr unsigned MINE = J * NB * 1024;
        char* const out = reinterpret_cast<char*>(part) + (size_t)tile * nks * WAVES * MINE;
        const __amdgpu_buffer_rsrc_t pr = w4_make_rsrc(out, (unsigned)nks * WAVES * MINE);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < NB; i++)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, acc[j][i]), pr, lane * 16, ((int)slice * WAVES + wave) * (int)MINE + (j * NB + i) * 1024, DEVICE);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) *last_one = __hip_atomic_fetch_add(tickets + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nks - 1;
        __syncthreads();
        if (!*last_one) return;
        if (threadIdx.x == 0) __hip_atomic_store(tickets + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < NB; i++) acc[j][i] = (f4_t){0.f, 0.f, 0.f, 0.f};
        for (int o = 0; o < nks; o++) {
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < NB; i++)
                    acc[j][i] += __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(pr, lane * 16, (o * WAVES + wave) * (int)MINE + (j * NB + i) * 1024, DEVICE));
        }
    }
    // D register e of lane (tok, kg): output column 4 kg + e of its row block, row tok
    constexpr int OUT = GLU ? NB / 2 : NB;
    const int c0 = wrb * 16 + kg * 4;
    auto store = [&](auto type) {
        constexpr int T = decltype(type)::value;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int m = m0 + j * 16 + tok;
            const size_t row_at = (size_t)m * out_n + c0;
#pragma unroll
            for (int i = 0; i < OUT; i++) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = GLU ? w4_act_mul(acc[j][i][e], acc[j][GLU ? i + OUT : i][e], act) : acc[j][i][e];
                if (m < t && c0 + i * 16 < out_n) w8_store4<T>(y, row_at + i * 16, out_n - c0 - i * 16, v);
            }
        }
    };
    // One type's code is run, and read for the first time: branches inside hold up the launch's end
    if (y_type == Q8_F32) store(w8_type<Q8_F32>{});
    else if (y_type == Q8_F16) store(w8_type<Q8_F16>{});
    else store(w8_type<Q8_BF16>{});
}

// What a workgroup of a tiled kernel has to do: a tile of BM rows and 64 NB columns of weights (gated: 32 NB outputs) and a k slice of it
template <int BM, int NB, bool GLU>
struct F8Tile {
    unsigned tile = 0, slice = 0;
    int out_n, m0 = 0, n0 = 0, wrb = 0, from = 0, to = 0;  // outputs, first row and output, first row block of the wave's columns, the slice's blocks of 128
    int x_rows = 0, w_rows[2] = {0, 0};            // row blocks of activations and of the wave's weights (gated: gate, values) that there are
    size_t w_first[2] = {0, 0};

    // false: nothing to do.  Every XCD takes a consecutive eighth of the tiles (and of their slices), bands of `band` tile rows, in a band m fastest
    __device__ __forceinline__ bool find(int wave, int n, int kb, int t, int nks, int band) {
        constexpr int BN = GLU ? NB * 32 : NB * 64, MINE = GLU ? NB / 2 : NB;
        const int half_rb = GLU ? n >> 5 : 0, w_end = GLU ? half_rb : (n + 15) >> 4;
        out_n = GLU ? n >> 1 : n;
        const int tiles_m = (t + BM - 1) / BM, tiles_n = (out_n + BN - 1) / BN;
        const unsigned work = (unsigned)tiles_m * (unsigned)tiles_n * (unsigned)nks, xcd = blockIdx.x & 7;
        const unsigned at = (unsigned)((unsigned long long)work * xcd / 8) + (blockIdx.x >> 3);
        if (at >= (unsigned)((unsigned long long)work * (xcd + 1) / 8)) return false;
        auto uniform = [](auto v) { return (decltype(v))__builtin_amdgcn_readfirstlane((int)v); };  // as all of this is: quotients come from the vector unit
        tile = uniform(at / (unsigned)nks);
        slice = at - tile * (unsigned)nks;
        const unsigned per_band = (unsigned)band * tiles_n, b_at = uniform(tile / per_band), in_band = tile - b_at * per_band;
        const unsigned rows = min((unsigned)band, (unsigned)tiles_m - b_at * band);
        const int tn = (int)uniform(in_band / rows), tm = (int)(b_at * band + in_band - tn * rows);
        m0 = tm * BM;
        x_rows = (int)uniform(min(((t + 15) >> 4) - (m0 >> 4), BM / 16));
        n0 = tn * BN;
        wrb = (n0 >> 4) + wave * MINE;
        w_rows[0] = w_rows[1] = (int)uniform(max(min(w_end - wrb, MINE), 0));
        w_first[0] = (unsigned)uniform(w_rows[0] ? wrb : 0);
        w_first[1] = GLU ? (size_t)half_rb + w_first[0] : w_first[0];
        from = (int)uniform((unsigned)kb * slice / (unsigned)nks);  // (at most 1024 blocks and 8 slices)
        to = (int)uniform((unsigned)kb * (slice + 1) / (unsigned)nks);
        return true;
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t x_rsrc(const char* x, int kb) const {
        return w4_make_rsrc(x + (size_t)(m0 >> 4) * kb * 2048, (unsigned)x_rows * (unsigned)kb * 2048u);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t w_rsrc(const char* w, int kb, int part) const {
        return w4_make_rsrc(w + w_first[part] * (unsigned)kb * 2048, (unsigned)w_rows[part] * (unsigned)kb * 2048u);
    }
    // One of the two rows of the weights' scales that the tile's columns lie in (gated: the gate's and the values'), and the one of a wave's columns
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t s_rsrc(const float* s, int n, int kb, int part) const {
        const int row = __builtin_amdgcn_readfirstlane(GLU ? (n0 >> 7) + part * (n >> 8) : min((n0 >> 7) + part, (n - 1) >> 7));
        return w4_make_rsrc(s + (size_t)row * kb, (unsigned)kb * 4u);
    }
    __device__ __forceinline__ static int s_part(int wave, int i) { return GLU ? i / (NB / 2) : wave * NB * 16 >> 7; }
    // Offset of row block i of the wave's weights (gated: the first half are the gate's, the second its values') and of the activations.
    // Behind the last one the last again, whose results are not stored: a load's scalar offset takes no part in its bounds check.
    __device__ __forceinline__ int w_row(int i, int kb) const {
        return __builtin_amdgcn_readfirstlane(max(min(GLU ? i % (NB / 2) : i, w_rows[0] - 1), 0) * kb * 2048);
    }
    __device__ __forceinline__ int x_row(int j, int kb) const { return __builtin_amdgcn_readfirstlane(min(j, x_rows - 1) * kb * 2048); }
};

// One block of 128 of 16 x 16 sums: weights (halves b), activations (halves a), without scales the plain form
__device__ __forceinline__ f4_t f8_product(u4_t b0, u4_t b1, u4_t a0, u4_t a1) {
    const i8_t b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
    const i8_t a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, (f4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// ------------------------------------------------------------------------------------------------ 64 x 128 tiles of e4m3 products
template <bool GLU>
__device__ __forceinline__ void f8_tiled_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                              const float* __restrict__ xs, void* __restrict__ y, int n, int kb, int t, int y_type, int act, int nks,
                                              int band, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int BM = 64, NB = 2, J = BM / 16, XL = J / 2;
    __shared__ __attribute__((aligned(1024))) char lds[2][BM * 128];  // a block of activations: [row block][k tile] of 1 KiB
    __shared__ float scale[2][2][BM];  // of rows and weights: their products, for the two rows of the weights' scales
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = lane & 15;
    F8Tile<BM, NB, GLU> T;
    if (!T.find(wave, n, kb, t, nks, band)) return;
    const int from = T.from, to = T.to;
    const __amdgpu_buffer_rsrc_t xr = T.x_rsrc(xq, kb), wr0 = T.w_rsrc(wt, kb, 0), wr1 = GLU ? T.w_rsrc(wt, kb, 1) : wr0;
    const unsigned at_lane = lane * 16u;
    int w_row[NB], x_row[XL];  // of the wave's weights, and of the row blocks of which it brings a k tile each: tile 4 i + wave of a block's 2 j + h
#pragma unroll
    for (int i = 0; i < NB; i++) w_row[i] = T.w_row(i, kb);
#pragma unroll
    for (int i = 0; i < XL; i++) x_row[i] = T.x_row(2 * i + (wave >> 1), kb) + (wave & 1) * 1024;
    u4_t w[2][NB][2], x[XL];
    float xs_next = 0.f, ws_next = 0.f;
    auto load_w = [&](u4_t& d, int k, int i, int h) {
        const int at = min(k, to - 1) * 2048 + h * 1024;  // behind the end the last block again, not used
        d = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(GLU && i >= NB / 2 ? wr1 : wr0, at_lane, w_row[i] + at, 0));
    };
    const int s_row = threadIdx.x % BM, s_part = __builtin_amdgcn_readfirstlane(threadIdx.x / BM & 1);  // of the scales, a product to each thread (BM = 64: two)
    const __amdgpu_buffer_rsrc_t sr = T.s_rsrc(ws, n, kb, s_part);
    const int xs_row = min(T.m0 + s_row, t - 1);
    auto load_x = [&](int k) {
        const int kk = min(k, to - 1);
#pragma unroll
        for (int i = 0; i < XL; i++) x[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(xr, at_lane, x_row[i] + kk * 2048, 0));
        xs_next = xs[(size_t)kk * t + xs_row];
        ws_next = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(sr, 0, kk * 4, 0));
    };
    auto put_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < XL; i++) *reinterpret_cast<u4_t*>(lds[buf] + (4 * i + wave) * 1024 + lane * 16) = x[i];
        scale[buf][s_part][s_row] = xs_next * ws_next;
    };
    f4_t acc[J][NB];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) acc[j][i] = (f4_t){0.f, 0.f, 0.f, 0.f};
    if (from < to) {
        load_x(from);
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) load_w(w[0][i][h], from, i, h);
        put_x(0);
        load_x(from + 1);
        w8_lds_done();
        w8_lds_barrier();
        for (int k = from;;) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int i = 0; i < NB; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) load_w(w[1 - u][i][h], k + 1, i, h);
                put_x(1 - u);  // block k + 1, asked for a block ago; the buffer was read last before the barrier
                load_x(k + 2);
#pragma unroll
                for (int j = 0; j < J; j++) {
                    f4_t p[NB];
                    const u4_t a0 = *reinterpret_cast<const u4_t*>(lds[u] + 2 * j * 1024 + lane * 16), a1 = *reinterpret_cast<const u4_t*>(lds[u] + (2 * j + 1) * 1024 + lane * 16);
#pragma unroll
                    for (int i = 0; i < NB; i++) p[i] = f8_product(w[u][i][0], w[u][i][1], a0, a1);
#pragma unroll
                    for (int i = 0; i < NB; i++) {
                        const float s = scale[u][T.s_part(wave, i)][j * 16 + tok];
                        acc[j][i] = w4_fma4(p[i], (f4_t){s, s, s, s}, acc[j][i]);
                    }
                }
                if (++k >= to) goto summed;
                w8_lds_done();
                w8_lds_barrier();
            }
        }
    }
summed:
    f8_finish<J, NB, GLU>(acc, &last_one, T.wrb, T.m0, T.out_n, t, y, y_type, act, nks, T.slice, T.tile, part, tickets);
}

// ------------------------------------------------------------------------------------------------ 128 x 256 tiles of e4m3 products
// The 128 sums a lane leave 128 registers: weights a block ahead (64), activations in halves of 8, into three LDS buffers, two blocks ahead, so that a block's first
// operands are read ahead of the barrier that ends the block before.  The order of loads, products and sums is written out: a product enters its sum three products later, when it is
// there, and no branch stands inside a block, behind which the compiler would wait for all loads in flight: 656 us at 4096 rows, 670 with a branch, 712 with one and sums at once.
template <bool GLU>
__device__ __forceinline__ void f8_wide_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq, const float* __restrict__ xs,
                                             void* __restrict__ y, int n, int kb, int t, int y_type, int act, int nks, int band, w8_pair_t* __restrict__ part,
                                             int* __restrict__ tickets) {
    constexpr int BM = 128, NB = 4, J = BM / 16, XL = J / 2;
    __shared__ __attribute__((aligned(1024))) char lds[3][BM * 128];  // a block of activations: [row block][k tile] of 1 KiB
    __shared__ float scale[3][2][BM];  // of rows and weights: their products, for the two rows of the weights' scales
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = lane & 15;
    F8Tile<BM, NB, GLU> T;
    if (!T.find(wave, n, kb, t, nks, band)) return;
    const int from = T.from, to = T.to;
    const __amdgpu_buffer_rsrc_t xr = T.x_rsrc(xq, kb), wr0 = T.w_rsrc(wt, kb, 0), wr1 = GLU ? T.w_rsrc(wt, kb, 1) : wr0;
    const unsigned at_lane = lane * 16u;
    int w_row[NB], x_row[XL];  // of the wave's weights, and of the row blocks of which it brings a k tile each: tile 4 i + wave of a block's 2 j + h
#pragma unroll
    for (int i = 0; i < NB; i++) w_row[i] = T.w_row(i, kb);
#pragma unroll
    for (int i = 0; i < XL; i++) x_row[i] = T.x_row(2 * i + (wave >> 1), kb) + (wave & 1) * 1024;
    u4_t w[2][NB][2], x[XL / 2], a[2][2];
    float xs_next = 0.f, ws_next = 0.f, sc[2][2];  // sc: read ahead as a is, gated with a second one
    auto load_w = [&](u4_t& d, int k, int i, int h) {
        const int at = min(k, to - 1) * 2048 + h * 1024;  // behind the end the last block again, not used
        d = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(GLU && i >= NB / 2 ? wr1 : wr0, at_lane, w_row[i] + at, 0));
    };
    const int s_row = threadIdx.x % BM, s_part = __builtin_amdgcn_readfirstlane(threadIdx.x / BM & 1);  // of the scales, a product to each thread (BM = 64: two)
    const __amdgpu_buffer_rsrc_t sr = T.s_rsrc(ws, n, kb, s_part);
    const int xs_row = min(T.m0 + s_row, t - 1);
    // half of a block's activations, 0 or 1; its scales come with the first
    auto load_x = [&](int k, int half) {
        const int kk = min(k, to - 1);
#pragma unroll
        for (int i = 0; i < XL / 2; i++)
            x[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(xr, at_lane, x_row[i + half * XL / 2] + kk * 2048, 0));
        if (half == 0) {
            xs_next = xs[(size_t)kk * t + xs_row];
            ws_next = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(sr, 0, kk * 4, 0));
        }
    };
    auto put_x = [&](int buf, int half) {
#pragma unroll
        for (int i = 0; i < XL / 2; i++) *reinterpret_cast<u4_t*>(lds[buf] + (4 * (i + half * XL / 2) + wave) * 1024 + lane * 16) = x[i];
        if (half == 0) scale[buf][s_part][s_row] = xs_next * ws_next;
    };
    auto get_a = [&](int buf, int j, int at) {
#pragma unroll
        for (int h = 0; h < 2; h++) a[at][h] = *reinterpret_cast<const u4_t*>(lds[buf] + (2 * j + h) * 1024 + lane * 16);
    };
    auto get_scales = [&](int buf, int j, int at) {
        sc[at][0] = scale[buf][T.s_part(wave, 0)][j * 16 + tok];
        if (GLU) sc[at][1] = scale[buf][1][j * 16 + tok];
    };
    f4_t acc[J][NB];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) acc[j][i] = (f4_t){0.f, 0.f, 0.f, 0.f};
    f4_t p[NB];  // products that are not in the sums yet
#pragma unroll
    for (int i = 0; i < NB; i++) p[i] = (f4_t){0.f, 0.f, 0.f, 0.f};
    if (from < to) {
        load_x(from, 0);
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) load_w(w[0][i][h], from, i, h);
        put_x(0, 0);
        load_x(from, 1);
        put_x(0, 1);
        load_x(from + 1, 0);
        put_x(1, 0);
        load_x(from + 1, 1);
        put_x(1, 1);
        load_x(from + 2, 0);
        w8_lds_done();
        w8_lds_barrier();
        get_a(0, 0, 0);
        get_scales(0, 0, 0);
        sc[1][0] = sc[1][1] = 0.f;
        // Leaving from the middle, not skipping steps: the compiler's waits count the loads of every way that leads to a step
        for (int k = from;;) {
#pragma unroll
            for (int u = 0; u < 6; u++) {  // weights alternate between two, activations between three
                const int cur = u & 1, buf = u % 3;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const u4_t a0 = a[j & 1][0], a1 = a[j & 1][1];
#pragma unroll
                    for (int i = 0; i < NB; i++) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (i == 0) {
                            if (j == 0) {
                                put_x((u + 2) % 3, 0);  // block k + 2, asked for half a block ago; the buffer was read last a block ago, which the barrier since then ends
                                load_x(k + 2, 1);
                            }
#pragma unroll
                            for (int q = 3 * j; q < min(3 * j + 3, 2 * NB); q++) load_w(w[1 - cur][q / 2][q & 1], k + 1, q / 2, q & 1);  // behind the activations that are waited for first
                            if (j == J / 2) {
                                put_x((u + 2) % 3, 1);
                                load_x(k + 3, 0);
                            }
                            if (j == J - 1) w8_lds_done();
                            if (j < J - 1) get_a(buf, j + 1, (j + 1) & 1);
                            else get_a((u + 1) % 3, 0, 0);  // written a block ago: there behind the last barrier
                        }
                        p[i] = f8_product(w[cur][i][0], w[cur][i][1], a0, a1);
                        __builtin_amdgcn_sched_barrier(0);
                        // the sum of three products ago: there, and its registers are the next product's
                        const int o = (i + 1) % NB, jo = i == NB - 1 ? j : (j + J - 1) % J;
                        const float f = sc[jo & 1][GLU ? o / (NB / 2) : 0];
                        acc[jo][o] = w4_fma4(p[o], (f4_t){f, f, f, f}, acc[jo][o]);
                        if (i == NB - 2) get_scales(j < J - 1 ? buf : (u + 1) % 3, (j + 1) % J, (j + 1) & 1);
                    }
                }
                w8_lds_barrier();
                if (++k >= to) goto summed;
            }
        }
    }
summed:
#pragma unroll
    for (int o = 1; o < NB; o++) {
        const float f = sc[1][GLU ? o / (NB / 2) : 0];
        acc[J - 1][o] = w4_fma4(p[o], (f4_t){f, f, f, f}, acc[J - 1][o]);
    }
    f8_finish<J, NB, GLU>(acc, &last_one, T.wrb, T.m0, T.out_n, t, y, y_type, act, nks, T.slice, T.tile, part, tickets);
}

// ------------------------------------------------------------------------------------------------ 64 x 128 and 64 x 256 tiles of f16 products
// A block is four chunks of 32 k.  A chunk's J NB products each continue a sum of the block, so that none waits for the one before it; beside each of them stands the conversion of
// a pair of weights for the next ones, and in a block's first chunk the addition of the sums of the block before.  Weights are in flight three halves of a block ahead, activations as in the
// wide kernel, as f16 in LDS (converted once, not by each wave).  All products of a row block in turn, its 64 weights converted ahead in one go: 1298 us, not 1214.
template <int NB, bool GLU>
__device__ __forceinline__ void f8_exact_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                              const float* __restrict__ xs, void* __restrict__ y, int n, int kb, int t, int y_type, int act, int nks,
                                              int band, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int BM = 64, J = BM / 16, XL = J / 2;
    static_assert(XL == 2 && J == 4, "a conversion of a pair beside each product");
    __shared__ __attribute__((aligned(1024))) char lds[3][BM * 256];  // a block of activations: [row block][chunk] of 1 KiB
    __shared__ float scale[3][2][BM];  // of rows and weights: their products, for the two rows of the weights' scales
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = lane & 15;
    F8Tile<BM, NB, GLU> T;
    if (!T.find(wave, n, kb, t, nks, band)) return;
    const int from = T.from, to = T.to;
    const __amdgpu_buffer_rsrc_t xr = T.x_rsrc(xq, kb), wr0 = T.w_rsrc(wt, kb, 0), wr1 = GLU ? T.w_rsrc(wt, kb, 1) : wr0;
    const unsigned at_lane = lane * 16u;
    int w_row[NB], x_row[XL];  // of the wave's weights, and of the row blocks of which it brings a k tile each: tile 4 i + wave of a block's 2 j + h
#pragma unroll
    for (int i = 0; i < NB; i++) w_row[i] = T.w_row(i, kb);
#pragma unroll
    for (int i = 0; i < XL; i++) x_row[i] = T.x_row(2 * i + (wave >> 1), kb) + (wave & 1) * 1024;
    u4_t w[3][NB], x;  // w: halves of blocks, the half 2 k + h in (2 k + h) % 3
    u4_t wh[2];  // 16 weights' eight k of a chunk, the next ones as well, and a chunk's activations with the next one's
    h8_t a[2][J];
    f4_t acc[J][NB], p[J][NB];
    float xs_next = 0.f, ws_next = 0.f, sc[J][2];  // sc: of the block whose sums are in p
    auto load_w = [&](u4_t& d, int k, int i, int h) {
        const int at = min(k, to - 1) * 2048 + h * 1024;  // behind the end the last block again, not used
        d = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(GLU && i >= NB / 2 ? wr1 : wr0, at_lane, w_row[i] + at, 0));
    };
    const int s_row = threadIdx.x % BM, s_part = __builtin_amdgcn_readfirstlane(threadIdx.x / BM & 1);  // of the scales, a product to each thread (BM = 64: two)
    const __amdgpu_buffer_rsrc_t sr = T.s_rsrc(ws, n, kb, s_part);
    const int xs_row = min(T.m0 + s_row, t - 1);
    auto load_x = [&](int k, int half) {
        const int kk = min(k, to - 1);
        x = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(xr, at_lane, x_row[half] + kk * 2048, 0));
        if (half == 0) {
            xs_next = xs[(size_t)kk * t + xs_row];
            ws_next = q8_f32(__builtin_amdgcn_raw_buffer_load_b32(sr, 0, kk * 4, 0));
        }
    };
    auto put_x = [&](int buf, int half) {
        char* const to_lds = lds[buf] + (4 * half + wave) * 2048 + lane * 16;
        *reinterpret_cast<h8_t*>(to_lds) = f8_to_f16(x[0], x[1]);
        *reinterpret_cast<h8_t*>(to_lds + 1024) = f8_to_f16(x[2], x[3]);
        if (half == 0) scale[buf][s_part][s_row] = xs_next * ws_next;
    };
    auto get_a = [&](int buf, int j, int c) { a[c & 1][j] = *reinterpret_cast<const h8_t*>(lds[buf] + (4 * j + c) * 1024 + lane * 16); };
    auto add = [&](int j, int i) {
        const float s = sc[j][GLU ? i / (NB / 2) : 0];
        acc[j][i] = w4_fma4(p[j][i], (f4_t){s, s, s, s}, acc[j][i]);
    };
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) acc[j][i] = p[j][i] = (f4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < J; j++) sc[j][0] = sc[j][1] = 0.f;
    if (from < to) {
        load_x(from, 0);
#pragma unroll
        for (int q = 0; q < 3; q++)
#pragma unroll
            for (int i = 0; i < NB; i++) load_w(w[q][i], from + q / 2, i, q & 1);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            put_x(b, 0);
            load_x(from + b, 1);
            put_x(b, 1);
            load_x(from + b + 1, 0);
        }
        wh[0] = __builtin_bit_cast(u4_t, f8_to_f16(w[0][0][0], w[0][0][1]));
        w8_lds_done();
        w8_lds_barrier();
#pragma unroll
        for (int j = 0; j < J; j++) get_a(0, j, 0);
        for (int k = from;;) {
#pragma unroll
            for (int u = 0; u < 3; u++) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
#pragma unroll
                    for (int i = 0; i < NB; i++) {
                        const int o = (i + 1) % NB, co = i == NB - 1 ? c + 1 : c, half = (2 * u + co / 2) % 3;  // the next products' weights, and where they are
#pragma unroll
                        for (int j = 0; j < J; j++) {
                            __builtin_amdgcn_sched_barrier(0);
                            if (c == 0) add(j, i);
                            p[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, wh[i & 1]), a[c & 1][j], c == 0 ? (f4_t){0.f, 0.f, 0.f, 0.f} : p[j][i], 0, 0, 0);
                            wh[o & 1][j] = f8_to_f16_pair(w[half][o][(co & 1) * 2 + j / 2], j & 1);
                            asm volatile("" : "+v"(wh[o & 1][j]));  // here, and not where it is used
                            if (i == 0) get_a(c < 3 ? u : (u + 1) % 3, j, (c + 1) & 3);  // behind the last barrier: written a block ago
                            if (c == 3 && i == 0) {
                                sc[j][0] = scale[u][T.s_part(wave, 0)][j * 16 + tok];
                                if (GLU) sc[j][1] = scale[u][1][j * 16 + tok];
                            }
                        }
                        if (co == 1 || co == 3) load_w(w[half][o], k + 1 + co / 2, o, 1 - co / 2);  // both of its chunks are converted: the half of a block three further on
                        if (c == 1 && i == 0) {  // block k + 2, asked for half a block ago; the buffer was read last a block ago, which the barrier since then ends
                            put_x((u + 2) % 3, 0);
                            load_x(k + 2, 1);
                        }
                        if (c == 3 && i == 0) {
                            put_x((u + 2) % 3, 1);
                            load_x(k + 3, 0);
                        }
                        if (c == 3 && i == NB - 1) w8_lds_done();  // what was written for block k + 2 is there, what was read of this one has been
                    }
                }
                w8_lds_barrier();
                if (++k >= to) goto summed;
            }
        }
    }
summed:
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) add(j, i);
    f8_finish<J, NB, GLU>(acc, &last_one, T.wrb, T.m0, T.out_n, t, y, y_type, act, nks, T.slice, T.tile, part, tickets);
}

#define F8_TILED(NAME, BODY, GLU)                                                                                                 \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                              int kb, int t, int y_type, int act, int nks, int band, w8_pair_t* part,  \
                                                              int* tickets) {                                                     \
        BODY<GLU>(wt, ws, xq, xs, y, n, kb, t, y_type, act, nks, band, part, tickets);                                          \
    }
#define F8_EXACT(NAME, NB, GLU)                                                                                                   \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                              int kb, int t, int y_type, int act, int nks, int band, w8_pair_t* part,  \
                                                              int* tickets) {                                                     \
        f8_exact_body<NB, GLU>(wt, ws, xq, xs, y, n, kb, t, y_type, act, nks, band, part, tickets);                             \
    }
F8_TILED(w4a16_f8_tiled_m64, f8_tiled_body, false)
F8_TILED(w4a16_f8_tiled_m64_glu, f8_tiled_body, true)
F8_TILED(w4a16_f8_tiled_m128, f8_wide_body, false)
F8_TILED(w4a16_f8_tiled_m128_glu, f8_wide_body, true)
F8_EXACT(w4a16_f8_exact_n128, 2, false)
F8_EXACT(w4a16_f8_exact_n128_glu, 2, true)
F8_EXACT(w4a16_f8_exact_n256, 4, false)
F8_EXACT(w4a16_f8_exact_n256_glu, 4, true)
