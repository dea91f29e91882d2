// FP8 linears:  y[m][n] = sum_b sx[b][m] * sw[n / 128][b] * sum_{k in b} q[m][k] w[n][k],  q and w e4m3 in tiles (q8_common.hpp, two k tiles
// to a block of 128), an f32 scale for each 128 k of a row and for each 128 x 128 of the weights.  A block's products are summed from zero on the matrix
// units and enter the running sum with one fused multiply-add.  Gated form: rows 0..n/2 of w are a gate, the rest its values, y[m][c] = act(gate) * value.
//
// Which product.  The e4m3 matrix instruction aligns products to the largest of their group and drops what lies 2^-14 and more below it: on normal
// numbers 1.6e-5 of the results' size, 4.2 PFLOP/s alone (16x16x128; 32x32x64 3.8), 3.5 with the scaling.  As f16, which holds every e4m3 number, the same
// sums are those of 32 bits (1e-8), at the f16 instruction's 1.6.  So: up to 64 rows, where the weight stream is what takes the time, and for f32 results, f16; for 16-bit
// results of more rows, whose own rounding is 30 times as large and whose rows' quantisation 1000 times, e4m3.
#include "f8_common.hpp"

typedef int i8_t __attribute__((ext_vector_type(8)));

// Eight e4m3 numbers as f16, exactly
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
// Up to 16 rows of floats (XT: their type) are quantised on the way: a wave takes of its run of k what it needs, once, behind its first weights; that is 16 conversions of eight
// cycles a lane and block, and saves the launch that would do it.
template <int XT>
struct F8Rows {  // a lane's share of a block of 16 activation rows, row lane % 16: chunks kg and kg + 4 of eight
    F8Run<XT> run[2];
    const char* row;
    int k, kg;
    __device__ __forceinline__ void at(const void* x, size_t ldx, int k_, int t) {
        row = static_cast<const char*>(x) + (size_t)min((int)(threadIdx.x & 15), t - 1) * ldx * (XT == Q8_F32 ? 4 : 2);
        k = k_;
        kg = (threadIdx.x & 63) >> 4;
    }
    __device__ __forceinline__ void load(int block) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int from = block * 128 + h * 64 + kg * 16;
            run[h].load(row, from, block * 128 + 128 <= k ? 16 : k - from);  // whole blocks without a branch
        }
    }
    // its e4m3 numbers as f16, and their scale
    __device__ __forceinline__ void get(h8_t (&x)[4], float& s) const {
        unsigned m = run[1].most(run[0].most(0));
        const auto a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        m = max(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
        m = max(b[0], b[1]);
        float by;
        s = f8_step(m, by);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const u4_t q = run[h].pack(by, !(s > 0.f));
            x[2 * h] = f8_to_f16(q[0], q[1]);
            x[2 * h + 1] = f8_to_f16(q[2], q[3]);
        }
    }
};
template <>
struct F8Rows<F8_ROWS> {};

template <int RB, int TT, bool GLU, int XT>
__device__ __forceinline__ void f8_skinny_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                               const float* __restrict__ xs, size_t ldx, int k_in, void* __restrict__ y, int n, int kb, int t, int R, int y_type,
                                               int act, int W, int nks, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr bool FLOATS = XT != F8_ROWS;
    static_assert(!FLOATS || TT == 1, "floats: up to 16 rows");
    constexpr int TILES = RB * TT, DEPTH = TILES == 1 ? (XT == Q8_F32 ? 3 : 4) : TILES <= 8 ? 2 : 1, SLOTS = TILES <= 4 ? 8 : 4, XD = FLOATS ? 1 : DEPTH;
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
    F8Rows<XT> rows;
    if constexpr (FLOATS) {
        rows.at(xq, ldx, k_in, t);
        if (lo < hi) rows.load(lo);
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
    const char* const xp = FLOATS ? nullptr : xq + ((size_t)kg * R + tok % R) * 16;
    const size_t x_tile = (size_t)R * 64, x_block = x_tile * 2 * kb;
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
            rows.load(k);
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
                if constexpr (FLOATS) {
                    rows.get(x[0], sx[0]);
                    if (k + d + 1 < hi) load_x(0, k + d + 1);
                } else {
#pragma unroll
                    for (int j = 0; j < TT; j++) {
                        sx[j] = xsv[d][j];
#pragma unroll
                        for (int c = 0; c < 4; c++) x[j][c] = f8_to_f16(xv[d][j][c / 2][c % 2 * 2], xv[d][j][c / 2][c % 2 * 2 + 1]);
                    }
                    if (next < hi) load_x(d, next);
                }
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
        for (int w = 0; w < adders; w++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += sums[w][tile][e][lane];
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
F8_SKINNY_T(w4a16_f8_skinny_r4, 4, false, )
F8_SKINNY_T(w4a16_f8_skinny_r2, 2, true, _glu)
F8_SKINNY_T(w4a16_f8_skinny_r4, 4, true, _glu)

// ------------------------------------------------------------------------------------------------ tiles, any number of rows
// Block tile BM = 64 or 128 rows x NB * 64 columns, four waves along n, wave tile BM x NB * 16.  Weights go straight into registers, a block ahead; activations
// and their scales through registers into LDS, two blocks ahead, of which there are two buffers: a block's barrier lets every wave read what was written during
// the block before.  EXACT: the activations become f16 on their way into LDS, the weights before their products.
// nks > 1: slices of k go to several workgroups, which hand their sums over as those of the kernels above do, added in the order of the slices.
template <int BM, int NB, bool EXACT, bool GLU>
__device__ __forceinline__ void f8_tiled_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                              const float* __restrict__ xs, void* __restrict__ y, int n, int kb, int t, int y_type, int act, int nks,
                                              int band, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int J = BM / 16, XL = J / 2, WAVES = 4, XB = EXACT ? 2 : 1;  // XB: bytes of an activation in LDS
    __shared__ __attribute__((aligned(1024))) char lds[2][BM * 128 * XB];  // a block of activations: [row block][k tile] of 1 KiB, or of 2
    __shared__ float x_scale[2][BM];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = lane & 15, kg = lane >> 4;
    const int out_n = GLU ? n >> 1 : n, half_rb = GLU ? n >> 5 : 0, row_blocks = (n + 15) >> 4;
    constexpr int BN = GLU ? NB * 32 : NB * 64;  // outputs
    // Block tiles: every XCD takes a consecutive eighth of them (and of their slices), bands of `band` tile rows, in a band m fastest
    const int tiles_m = (t + BM - 1) / BM, tiles_n = (out_n + BN - 1) / BN;
    const unsigned work = (unsigned)tiles_m * (unsigned)tiles_n * (unsigned)nks, xcd = blockIdx.x & 7;
    const unsigned at = (unsigned)((unsigned long long)work * xcd / 8) + (blockIdx.x >> 3);
    if (at >= (unsigned)((unsigned long long)work * (xcd + 1) / 8)) return;
    const unsigned tile = at / (unsigned)nks, slice = at - tile * (unsigned)nks;
    const unsigned per_band = (unsigned)band * tiles_n, b_at = tile / per_band, in_band = tile - b_at * per_band;
    const unsigned rows = min((unsigned)band, (unsigned)tiles_m - b_at * band);
    const int tn = (int)(in_band / rows), tm = (int)(b_at * band + in_band - tn * rows);
    const int m0 = tm * BM, n0 = tn * BN;

    const int x_blocks = (t + 15) >> 4;
    const __amdgpu_buffer_rsrc_t xr = w4_make_rsrc(xq + (size_t)(m0 >> 4) * kb * 2048, (unsigned)min(x_blocks - (m0 >> 4), J) * (unsigned)kb * 2048u);
    // first row block of the wave's columns and what is left of the matrix behind it
    const int wrb = (n0 >> 4) + wave * (GLU ? NB / 2 : NB), w_end = GLU ? half_rb : row_blocks;
    auto w_rsrc = [&](int first, int count) {
        first = __builtin_amdgcn_readfirstlane(count > 0 ? first : 0);  // uniform, and known to be
        count = __builtin_amdgcn_readfirstlane(max(count, 0));
        return w4_make_rsrc(wt + (size_t)(unsigned)first * (unsigned)kb * 2048, (unsigned)count * (unsigned)kb * 2048u);
    };
    const __amdgpu_buffer_rsrc_t wr0 = w_rsrc(wrb, min(w_end - wrb, GLU ? NB / 2 : NB)),
                                 wr1 = GLU ? w_rsrc(half_rb + wrb, min(w_end - wrb, NB / 2)) : wr0;
    // The wave's columns lie in one row of the weights' scales (gated: one of the gate's, one of the values')
    const float* const ws0 = ws + (size_t)(min(wrb, w_end - 1) >> 3) * kb;
    const float* const ws1 = GLU ? ws + (size_t)((half_rb + min(wrb, w_end - 1)) >> 3) * kb : ws0;
    // row block slot i of the wave: gated, the first half are the gate's, the second its values'
    unsigned wo[NB], xo[XL];
#pragma unroll
    for (int i = 0; i < NB; i++) wo[i] = (unsigned)(GLU ? i % (NB / 2) : i) * (unsigned)kb * 2048u + lane * 16u;
    // activations: 1 KiB tiles 2 j + h of a block (row block j, k tile h), tile 4 i + wave to this wave
#pragma unroll
    for (int i = 0; i < XL; i++) xo[i] = (unsigned)(2 * i + (wave >> 1)) * (unsigned)kb * 2048u + (wave & 1) * 1024u + lane * 16u;
    const int from = (int)((long long)kb * slice / nks), to = (int)((long long)kb * (slice + 1) / nks);
    u4_t w[2][NB][2], x[XL];
    float xs_next = 0.f;
    auto load_w = [&](u4_t (&d)[NB][2], int k) {
        const int at = min(k, to - 1) * 2048;  // behind the end the last block again, not used
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) d[i][h] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(GLU && i >= NB / 2 ? wr1 : wr0, wo[i], at + h * 1024, 0));
    };
    const int xs_row = min(m0 + (int)threadIdx.x % BM, t - 1);
    auto load_x = [&](int k) {
        const int kk = min(k, to - 1);
#pragma unroll
        for (int i = 0; i < XL; i++) x[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(xr, xo[i], kk * 2048, 0));
        xs_next = xs[(size_t)kk * t + xs_row];
    };
    auto put_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < XL; i++) {
            if (EXACT) {
                char* const p = lds[buf] + (4 * i + wave) * 2048 + lane * 16;
                *reinterpret_cast<h8_t*>(p) = f8_to_f16(x[i][0], x[i][1]);
                *reinterpret_cast<h8_t*>(p + 1024) = f8_to_f16(x[i][2], x[i][3]);
            } else {
                *reinterpret_cast<u4_t*>(lds[buf] + (4 * i + wave) * 1024 + lane * 16) = x[i];
            }
        }
        if (threadIdx.x < BM) x_scale[buf][threadIdx.x] = xs_next;
    };
    f4_t acc[J][NB];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) acc[j][i] = (f4_t){0.f, 0.f, 0.f, 0.f};
    float wsv0 = 0.f, wsv1 = 0.f;
    int base = from - 64;  // of the 64 blocks whose scales are in the lanes: none yet
    auto step = [&](const u4_t (&wv)[NB][2], int buf, int k) {
        if (k >= base + 64) {
            base = k;
            wsv0 = ws0[min(base + lane, kb - 1)];
            wsv1 = GLU ? ws1[min(base + lane, kb - 1)] : wsv0;
        }
        const float sw0 = f8_lane(wsv0, k - base), sw1 = GLU ? f8_lane(wsv1, k - base) : sw0;
        h8_t wh[EXACT ? NB : 1][4];
        if (EXACT) {
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) wh[EXACT ? i : 0][c] = f8_to_f16(wv[i][c / 2][c % 2 * 2], wv[i][c / 2][c % 2 * 2 + 1]);
        }
#pragma unroll
        for (int j = 0; j < J; j++) {
            f4_t p[NB];
            if (EXACT) {
                h8_t a[4];
#pragma unroll
                for (int c = 0; c < 4; c++) a[c] = *reinterpret_cast<const h8_t*>(lds[buf] + (2 * j + c / 2) * 2048 + (c & 1) * 1024 + lane * 16);
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < NB; i++)
                        p[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[EXACT ? i : 0][c], a[c], c == 0 ? (f4_t){0.f, 0.f, 0.f, 0.f} : p[i], 0, 0, 0);
            } else {
                const u4_t a0 = *reinterpret_cast<const u4_t*>(lds[buf] + 2 * j * 1024 + lane * 16), a1 = *reinterpret_cast<const u4_t*>(lds[buf] + (2 * j + 1) * 1024 + lane * 16);
                const i8_t a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
#pragma unroll
                for (int i = 0; i < NB; i++) {
                    const i8_t b = {(int)wv[i][0][0], (int)wv[i][0][1], (int)wv[i][0][2], (int)wv[i][0][3], (int)wv[i][1][0], (int)wv[i][1][1], (int)wv[i][1][2], (int)wv[i][1][3]};
                    p[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, (f4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);  // no scales: the plain form
                }
            }
            const float sx = x_scale[buf][j * 16 + tok], s0 = sx * sw0, s1 = GLU ? sx * sw1 : s0;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const float s = GLU && i >= NB / 2 ? s1 : s0;
                acc[j][i] = w4_fma4(p[i], (f4_t){s, s, s, s}, acc[j][i]);
            }
        }
    };
    if (from < to) {
        load_x(from);
        load_w(w[0], from);
        put_x(0);
        load_x(from + 1);
        __syncthreads();
        for (int k = from;;) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                load_w(w[1 - u], k + 1);
                put_x(1 - u);  // block k + 1, asked for a block ago; the buffer was read last before the barrier
                load_x(k + 2);
                step(w[u], u, k);
                if (++k >= to) goto summed;
                w8_lds_done();
                w8_lds_barrier();
            }
        }
    }
summed:
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
        if (threadIdx.x == 0) last_one = __hip_atomic_fetch_add(tickets + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nks - 1;
        __syncthreads();
        if (!last_one) return;
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

#define F8_TILED(NAME, BM, NB, EXACT, GLU)                                                                                        \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                              int kb, int t, int y_type, int act, int nks, int band, w8_pair_t* part,  \
                                                              int* tickets) {                                                     \
        f8_tiled_body<BM, NB, EXACT, GLU>(wt, ws, xq, xs, y, n, kb, t, y_type, act, nks, band, part, tickets);                    \
    }
F8_TILED(w4a16_f8_tiled_m64, 64, 4, false, false)
F8_TILED(w4a16_f8_tiled_m64_glu, 64, 4, false, true)
F8_TILED(w4a16_f8_tiled_m64_n128, 64, 2, false, false)
F8_TILED(w4a16_f8_tiled_m64_n128_glu, 64, 2, false, true)
F8_TILED(w4a16_f8_exact_m64, 64, 4, true, false)
F8_TILED(w4a16_f8_exact_m64_glu, 64, 4, true, true)
F8_TILED(w4a16_f8_exact_m64_n128, 64, 2, true, false)
F8_TILED(w4a16_f8_exact_m64_n128_glu, 64, 2, true, true)
