// W8A8 linears:  y[m][n] = (sum_k q[m][k] w[n][k]) * s[m] * ws[n],  q and w int8 in tiles (q8_common.hpp), sums in 32-bit whole
// numbers (exact: k <= 131071), one f32 scale per row of either.  Gated form: rows 0..n/2 of w are a gate, the rest its values,
// y[m][c] = act(gate) * value, [t][n/2].
#include "q8_common.hpp"

// y[at .. at + 3] (those below `left`) as f32, f16 or bf16
template <int T>
__device__ __forceinline__ void w8_store4(void* __restrict__ y, size_t at, int left, const float (&v)[4]) {
    if (T == Q8_F32) {
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
    for (int i = 0; i < 4; i++) h[i] = q8_to_16<T>(v[i]);
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
__device__ __forceinline__ void w8_store4(void* __restrict__ y, size_t at, int left, const float (&v)[4], int y_type) {
    if (y_type == Q8_F32) w8_store4<Q8_F32>(y, at, left, v);
    else if (y_type == Q8_F16) w8_store4<Q8_F16>(y, at, left, v);
    else w8_store4<Q8_BF16>(y, at, left, v);
}

// ------------------------------------------------------------------------------------------------ up to 64 rows
// The weight stream bounds these launches.  A workgroup's waves, two at least, take consecutive runs of a k slice of the same RB row blocks (16
// outputs each); the weights arrive as whole tiles straight in registers, DEPTH of them in flight per row block, meet TT tiles of 16
// activation rows (from the L2), and the waves' sums are added in LDS: whole numbers, so in any order the same.  Where there are too
// few row blocks for the chip, slices of k go to several workgroups (gridDim.y of them): each leaves its sums in the workspace and
// draws a ticket of its row blocks, the last one adds them.  More than TT * 16 rows: groups of so many, each through all of it.
// Launches back to back: 34816 x 5120 gated at t = 1 31.5 us (5.7 TB/s), 131072 x 5120 at t = 4 98 us (6.8), where a library's sum reads at 6.0 and a
// copy moves 5.1; 4096 x 4096 at t = 1 5.2 us, of which about 2 are the launch's way to its first weights.
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

    const int ks = blockIdx.y % (unsigned)nks, group = blockIdx.y / (unsigned)nks, groups = gridDim.y / (unsigned)nks;
    const int runs = nks * W, run = ks * W + wave;
    const int m0 = group * TT * 16, x_last = (t - 1) >> 4;  // rows of the group, and the last tile of 16 that there is
    const int lo = (int)((long long)kt * run / runs), hi = (int)((long long)kt * (run + 1) / runs);
    i4_t acc[RB][TT];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) acc[i][j] = (i4_t){0, 0, 0, 0};
    i4_t wv[DEPTH][RB], xv[DEPTH][TT];
    auto load = [&](int d, int k) {
        // Non-temporal weights: 34816 x 5120 gated at t = 1 31.3 us, else 35.2; 4096 x 4096 at t = 128 in two groups 9.7, else 9.9
#pragma unroll
        for (int i = 0; i < RB; i++) wv[d][i] = __builtin_nontemporal_load(reinterpret_cast<const i4_t*>(wp[i] + (size_t)k * 1024));
#pragma unroll
        for (int j = 0; j < TT; j++) xv[d][j] = *reinterpret_cast<const i4_t*>(xp + min((m0 >> 4) + j, x_last) * x_block + k * x_tile);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (lo + d < hi) load(d, lo + d);
    for (int i = threadIdx.x; i < TILES * 256; i += W * 64) (&sums[0][0][0])[i] = 0;
    __syncthreads();
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
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < TT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                __hip_atomic_fetch_add(&sums[i * TT + j][e][lane], acc[i][j][e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    // A wave finishes every W-th tile (gated: a gate and its values)
    auto total = [&](int tile) {
        i4_t v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = sums[tile][e][lane];
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
            const i4_t v = total(u);
            w8_pair_t* const p = mine + ks * slice + u * 128;
            __hip_atomic_store(p, (w8_pair_t)(unsigned)v[1] << 32 | (unsigned)v[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(p + 64, (w8_pair_t)(unsigned)v[3] << 32 | (unsigned)v[2], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
// Block tile BM = 64 or 128 rows x NB * 64 = 128 or 256 columns, four waves along n, wave tile BM x NB * 16 on v_mfma_i32_16x16x64_i8 (the 32 x 32 x 32 form
// keeps up 3.3 POP/s on random bytes, this one 4.1).  Weights go straight into registers, activations through registers into LDS, a k tile
// of 64 at a time, both asked for AHEAD k tiles ahead: a line's first reader of an XCD waits up to 2 us for it.  Nothing waits for the
// newest loads: a k tile's barrier orders LDS alone, and with three LDS buffers the next tile's first blocks are read ahead of it.  The
// scales are fetched with the first tiles and the results' type is chosen once, or the tile's end took half as long as its products.
// 34816 x 5120 gated at t = 4096, launches back to back: 632 us, 2.3 POP/s of int8 (a library's product of this size without activation or scales
// 796); 604 to 736 in traces, by the clock that the power limit leaves.  The matrix units are busy 63 % of the time.  On a card where this took 591: LDS
// DMA, whose barriers have to wait for every load of the wave, 672; 650 with scales fetched at the end; with the loads one by one between the products
// within 3 % of this, both ways.
// nks > 1: slices of k go to several workgroups, which hand their sums over as those of the kernels above do.
template <int T>
struct w8_type {
    static constexpr int value = T;
};
__device__ __forceinline__ void w8_lds_done() { __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local"); }  // global loads stay in flight
__device__ __forceinline__ void w8_lds_barrier() {  // behind w8_lds_done
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int BM, int NB, int AHEAD, int XRING, bool GLU>
__device__ __forceinline__ void tiled_body(const char* __restrict__ wt, const float* __restrict__ ws, const char* __restrict__ xq,
                                           const float* __restrict__ xs, void* __restrict__ y, int n, int kt, int t, int y_type, int act, int nks,
                                           int band, w8_pair_t* __restrict__ part, int* __restrict__ tickets) {
    constexpr int J = BM / 16, XL = J / 4, WAVES = 4, PERIOD = XRING == AHEAD ? AHEAD * (AHEAD + 1) : AHEAD + 1;
    static_assert(BM % 64 == 0 && PERIOD % 3 == 0 && (XRING == AHEAD || XRING == AHEAD + 1), "rings and the three buffers fit the period");
    __shared__ __attribute__((aligned(1024))) char lds[3][BM * 64];  // a k tile of activations: [row block] of 1 KiB
    __shared__ __attribute__((aligned(16))) float w_scale[NB * 64], x_scale[BM];
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
    const __amdgpu_buffer_rsrc_t xr = w4_make_rsrc(xq + (size_t)(m0 >> 4) * kt * 1024, (unsigned)min(x_blocks - (m0 >> 4), BM / 16) * (unsigned)kt * 1024u);
    // first row block of the wave's columns and what is left of the matrix behind it
    const int wrb = (n0 >> 4) + wave * (GLU ? NB / 2 : NB), w_end = GLU ? half_rb : row_blocks;
    auto w_rsrc = [&](int first, int count) {
        first = __builtin_amdgcn_readfirstlane(count > 0 ? first : 0);  // uniform, and known to be
        count = __builtin_amdgcn_readfirstlane(max(count, 0));
        return w4_make_rsrc(wt + (size_t)(unsigned)first * (unsigned)kt * 1024, (unsigned)count * (unsigned)kt * 1024u);
    };
    const __amdgpu_buffer_rsrc_t wr0 = w_rsrc(wrb, min(w_end - wrb, GLU ? NB / 2 : NB)),
                                 wr1 = GLU ? w_rsrc(half_rb + wrb, min(w_end - wrb, NB / 2)) : wr0;
    // row block slot i of the wave: gated, the first half are the gate's, the second its values'
    unsigned wo[NB], xo[XL];
#pragma unroll
    for (int i = 0; i < NB; i++) wo[i] = (unsigned)(GLU ? i % (NB / 2) : i) * (unsigned)kt * 1024u + lane * 16u;
#pragma unroll
    for (int i = 0; i < XL; i++) xo[i] = (unsigned)(wave + 4 * i) * (unsigned)kt * 1024u + lane * 16u;
    const int from = (int)((long long)kt * slice / nks), to = (int)((long long)kt * (slice + 1) / nks);
    i4_t w[AHEAD + 1][NB], x[XRING][XL], a[4];  // k tiles i .. i + AHEAD of the weights, i + 2 .. i + AHEAD + 1 of the activations
    auto load_w = [&](i4_t (&d)[NB], int k) {
        const int at = min(k, to - 1) * 1024;  // behind the end the last tile again, not used
#pragma unroll
        for (int i = 0; i < NB; i++) d[i] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(GLU && i >= NB / 2 ? wr1 : wr0, wo[i], at, 0));
    };
    auto load_x = [&](i4_t (&d)[XL], int k) {
        const int at = min(k, to - 1) * 1024;
#pragma unroll
        for (int i = 0; i < XL; i++) d[i] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(xr, xo[i], at, 0));
    };
    auto put_x = [&](const i4_t (&s)[XL], int buf) {
#pragma unroll
        for (int i = 0; i < XL; i++) *reinterpret_cast<i4_t*>(lds[buf] + (wave + 4 * i) * 1024 + lane * 16) = s[i];
    };
    auto get_x = [&](int buf, int j) { return *reinterpret_cast<const i4_t*>(lds[buf] + j * 1024 + lane * 16); };
    i4_t acc[J][NB];
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int i = 0; i < NB; i++) acc[j][i] = (i4_t){0, 0, 0, 0};
    if (from < to) {
        i4_t first[XL];
        // the tile's scales, for its end: gated, first those of the gate, then of its values
        const int c = n0 + (int)(GLU ? threadIdx.x % BN : threadIdx.x), m = m0 + (int)threadIdx.x;
        const float cs = threadIdx.x < NB * 64 && c < out_n ? ws[GLU && threadIdx.x >= BN ? out_n + c : c] : 0.f, ms = threadIdx.x < BM && m < t ? xs[m] : 0.f;
        load_x(first, from);
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            load_x(x[(u + 1) % XRING], from + u + 1);
            load_w(w[u], from + u);
            __builtin_amdgcn_sched_barrier(0);  // in the order of the loop, whose waits count them
        }
        if (threadIdx.x < NB * 64) w_scale[threadIdx.x] = cs;
        if (threadIdx.x < BM) x_scale[threadIdx.x] = ms;
        put_x(first, 0);
        put_x(x[1], 1);
        w8_lds_done();
        w8_lds_barrier();
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = get_x(0, j);
        // Leaving from the middle, not skipping steps: the compiler's waits count the loads of every way that leads to a step
        for (int k = from;; k += PERIOD) {
#pragma unroll
            for (int u = 0; u < PERIOD; u++) {
                // k tile k + u from lds[u % 3], its first blocks in a; x holds tiles k + u + 2 .. k + u + AHEAD
                load_x(x[(u + AHEAD + 1) % XRING], k + u + AHEAD + 1);
                load_w(w[(u + AHEAD) % (AHEAD + 1)], k + u + AHEAD);
#pragma unroll
                for (int j = 0; j < J; j++) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (j == J / 2 - (J == 4 ? 2 : 1)) put_x(x[(u + 2) % XRING], (u + 2) % 3);  // read last a tile ago, which the barrier since then ends
#pragma unroll
                    for (int i = 0; i < NB; i++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u % (AHEAD + 1)][i], a[j & 3], acc[j][i], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (j == J - 4) w8_lds_done();
                    a[j & 3] = j < J - 4 ? get_x(u % 3, j + 4) : get_x((u + 1) % 3, j + 4 - J);  // written a tile ago: there behind the last barrier
                }
                w8_lds_barrier();
                if (k + u + 1 >= to) goto summed;
            }
        }
    }
summed:
    if (nks > 1) {
        // [tile][slice][wave][block of 16 x 16][64 lanes] of 16 bytes, at device scope: past this XCD's L2
        constexpr int DEVICE = 16;  // sc1
        constexpr unsigned MINE = J * NB * 1024;
        char* const base = reinterpret_cast<char*>(part) + (size_t)tile * nks * WAVES * MINE;
        const __amdgpu_buffer_rsrc_t pr = w4_make_rsrc(base, (unsigned)nks * WAVES * MINE);
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
        for (int o = 0; o < nks; o++) {
            if (o == (int)slice) continue;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < NB; i++)
                    acc[j][i] += __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(pr, lane * 16, (o * WAVES + wave) * (int)MINE + (j * NB + i) * 1024, DEVICE));
        }
    }
    // D register e of lane (tok, kg): output column 4 kg + e of its row block, row tok
    constexpr int OUT = GLU ? NB / 2 : NB;
    f4_t col[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) col[i] = *reinterpret_cast<const f4_t*>(&w_scale[(GLU ? i / OUT * BN : 0) + wave * OUT * 16 + i % OUT * 16 + kg * 4]);
    const int c0 = wrb * 16 + kg * 4;
    auto store = [&](auto type) {
        constexpr int T = decltype(type)::value;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int m = m0 + j * 16 + tok;
            const float sx = x_scale[j * 16 + tok];
            const size_t at = (size_t)m * out_n + c0;
#pragma unroll
            for (int i = 0; i < OUT; i++) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[e] = (float)acc[j][i][e] * sx * col[i][e];
                    if (GLU) v[e] = w4_act_mul(v[e], (float)acc[j][i + OUT][e] * sx * col[i + OUT][e], act);
                }
                if (m < t && c0 + i * 16 < out_n) w8_store4<T>(y, at + i * 16, out_n - c0 - i * 16, v);
            }
        }
    };
    // One type's code is run, and read for the first time: branches inside held up the launch's end
    if (y_type == Q8_F32) store(w8_type<Q8_F32>{});
    else if (y_type == Q8_F16) store(w8_type<Q8_F16>{});
    else store(w8_type<Q8_BF16>{});
}

#define W8_TILED(NAME, BM, NB, AHEAD, XRING, GLU)                                                                                 \
    extern "C" __global__ __launch_bounds__(256, 2) void NAME(const char* wt, const float* ws, const char* xq, const float* xs, void* y, int n, \
                                                              int kt, int t, int y_type, int act, int nks, int band, w8_pair_t* part,  \
                                                              int* tickets) {                                                     \
        tiled_body<BM, NB, AHEAD, XRING, GLU>(wt, ws, xq, xs, y, n, kt, t, y_type, act, nks, band, part, tickets);                \
    }
W8_TILED(w4a16_w8a8_tiled_m128, 128, 4, 3, 3, false)
W8_TILED(w4a16_w8a8_tiled_m128_glu, 128, 4, 3, 3, true)
W8_TILED(w4a16_w8a8_tiled_m64, 64, 4, 5, 6, false)
W8_TILED(w4a16_w8a8_tiled_m64_glu, 64, 4, 5, 6, true)
W8_TILED(w4a16_w8a8_tiled_m64_n128, 64, 2, 8, 9, false)
W8_TILED(w4a16_w8a8_tiled_m64_n128_glu, 64, 2, 8, 9, true)
