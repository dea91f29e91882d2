// Scoring of rows of logits z[V]: the log probability of a given token, the entropy of the distribution, and the most likely
// tokens with theirs.  One pass over the row with a running maximum:
//   S = sum 2^(z L - r),  U = sum (z L - r) 2^(z L - r),  L = log2 e, r = fl(max z * L), each term one fused multiply-add;
//   log p_j = ln 2 * ((z_j L - r) - log2 S),  entropy = ln 2 * (log2 S - U / S).
// r is the same rounded number in every term, so its rounding cancels; where z L could leave f32 (beyond 1e38: the lowest value of a
// type as a mask) the difference is taken before the factor.  A row that holds NaN or +infinity has NaN for all its
// numbers; a row of -infinity alone gives its tokens -infinity and the entropy 0.
//
// The best tokens: an element is the key (order-preserving image of its value << 32 | ~index), so that no two are alike and equal
// values rank by index.  Every wave keeps its candidates and a key that at least top_k of them exceed (or equal); an
// element is looked at only where its lane's maximum reaches that key's value.  Where more lanes than top_k reach it, it is raised
// first, to the top_k-th largest of the lanes' maxima: then at most 16 top_k elements are left.
// A row goes to one workgroup or, where there are few rows, to several: each leaves its record in the workspace and draws a
// ticket, the last one joins them.
#include "q8_common.hpp"

#define SCORE_MAX_TOP 32
#define SCORE_STAGE 1024       // elements of a wave's stage, 16 per lane
#define SCORE_WAVES 4
#define SCORE_CAP 576          // candidates of a wave: 64 carried over, 16 * SCORE_MAX_TOP of one stage
#define SCORE_RECORD 272       // bytes of a workgroup's record: max, S, U, padding, SCORE_MAX_TOP keys

typedef unsigned long long key_t_;

struct ScoreStats {
    float m, s, u;  // largest logit, S and U relative to fl(m * L)
};

__device__ __forceinline__ float score_ref(float m) { return m * 1.44269504088896341f; }
#define SCORE_BIG 1e38f
// ref(a) - ref(b) for a <= b; numbers so large that ref overflows are either equal or worlds apart
__device__ __forceinline__ float score_ref_diff(float a, float b) { return a == b ? 0.f : __builtin_fmaxf(score_ref(a) - score_ref(b), -1e30f); }
__device__ __forceinline__ float score_exp2(float d) { return __builtin_amdgcn_exp2f(d); }

// Sums relative to one maximum, re-expressed relative to a larger one and added.  -infinity: nothing there yet.
__device__ __forceinline__ ScoreStats score_join(ScoreStats a, ScoreStats b) {
    ScoreStats o;
    o.m = __builtin_elementwise_maximum(a.m, b.m);  // a NaN stays
    const float da = a.s > 0.f ? score_ref_diff(a.m, o.m) : 0.f, db = b.s > 0.f ? score_ref_diff(b.m, o.m) : 0.f;
    const float fa = score_exp2(da), fb = score_exp2(db);
    o.s = a.s * fa + b.s * fb;
    const float ua = a.u + a.s * da, ub = b.u + b.s * db;
    o.u = (fa > 0.f ? ua * fa : 0.f) + (fb > 0.f ? ub * fb : 0.f);
    return o;
}

__device__ __forceinline__ ScoreStats score_wave_join(ScoreStats a) {
#pragma unroll
    for (int st = 1; st < 64; st <<= 1) {
        ScoreStats b;
        b.m = __shfl_xor(a.m, st);
        b.s = __shfl_xor(a.s, st);
        b.u = __shfl_xor(a.u, st);
        // the same operands in the same order in both lanes: the same bits in every lane
        a = (threadIdx.x & st) ? score_join(b, a) : score_join(a, b);
    }
    return a;
}

__device__ __forceinline__ key_t_ score_key(float v, unsigned index) {
    const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);  // -0 ranks as 0
    const unsigned o = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (key_t_)o << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float score_value(key_t_ k) {
    const unsigned o = (unsigned)(k >> 32);
    return __builtin_bit_cast(float, (o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned score_index(key_t_ k) { return 0xffffffffu - (unsigned)k; }

__device__ __forceinline__ key_t_ score_lane(key_t_ v, int lane) {
    return (key_t_)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ void score_wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The candidates of one wave.  Everything here is uniform for the wave but the keys themselves.
struct ScoreTop {
    key_t_* buf;   // LDS, SCORE_CAP
    key_t_* out;   // LDS, SCORE_MAX_TOP
    int top, count;
    key_t_ low;    // an element has to exceed it; 0 is below every key

    __device__ __forceinline__ float floor_value() const { return low == 0 ? -__builtin_inff() : score_value(low); }

    // keeps the `top` best, best first
    __device__ void compact() {
        const int lane = threadIdx.x & 63;
        score_wave_sync();
        if (lane < SCORE_MAX_TOP) out[lane] = 0;
        score_wave_sync();
        for (int i = 0; i < count; i += 64) {
            const key_t_ mine = i + lane < count ? buf[i + lane] : 0;
            int rank = 0;
            for (int e = 0; e < count; e++) rank += buf[e] > mine;
            if (mine != 0 && rank < top) out[rank] = mine;
        }
        score_wave_sync();
        count = min(count, top);
        if (lane < count) buf[lane] = out[lane];
        score_wave_sync();
        if (count == top) {
            const key_t_ last = out[top - 1];
            low = max(low, score_lane(last, 0));
        }
    }

    // sixteen more keys per lane, 0 where there is none
    __device__ void take(const key_t_ (&key)[16]) {
        const int lane = threadIdx.x & 63;
        key_t_ best = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) best = max(best, key[j]);
        const unsigned long long over = __ballot(best > low);
        if (over == 0) return;
        if (__popcll(over) > top) {
            int rank = 0;
            for (int l = 0; l < 64; l++) rank += score_lane(best, l) > best;
            const unsigned long long at = __ballot(rank == top - 1 && best != 0);
            if (at) low = max(low, score_lane(best, __ffsll(at) - 1) - 1);
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const unsigned long long in = __ballot(key[j] > low);
            if (in == 0) continue;
            if (key[j] > low) buf[count + __builtin_amdgcn_mbcnt_hi((unsigned)(in >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)in, 0))] = key[j];
            count += __popcll(in);
        }
        if (count > 64) compact();
    }
};

// Raw 16 elements of a lane: element e is index at(e) of the stage
template <int T>
struct ScoreChunk {
    u4_t w[T == Q8_F32 ? 4 : 2];

    static __device__ __forceinline__ int at(int lane, int e) {
        return T == Q8_F32 ? (e >> 2) * 256 + lane * 4 + (e & 3) : (e >> 3) * 512 + lane * 8 + (e & 7);
    }
    // z: the row, first: its element the stage begins with, end: one past the last element of the row.  Elements behind it read as -infinity.
    __device__ __forceinline__ void load(const void* z, long long first, long long end, int lane) {
        constexpr int PER = T == Q8_F32 ? 4 : 8, N = T == Q8_F32 ? 4 : 2;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const long long i = first + at(lane, j * PER);
            if (i + PER <= end) {
                w[j] = *reinterpret_cast<const u4_any_t*>(static_cast<const char*>(z) + i * (T == Q8_F32 ? 4 : 2));
            } else {
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    if (T == Q8_F32) {
                        w[j][d] = i + d < end ? static_cast<const unsigned*>(z)[i + d] : 0xff800000u;
                    } else {
                        const unsigned none = T == Q8_F16 ? 0xfc00u : 0xff80u;
                        const uint16_t* const h = static_cast<const uint16_t*>(z);
                        w[j][d] = (i + 2 * d < end ? h[i + 2 * d] : none) | (i + 2 * d + 1 < end ? h[i + 2 * d + 1] : none) << 16;
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[16]) const {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (T == Q8_F32) v[e] = q8_f32(w[e >> 2][e & 3]);
            else if (T == Q8_F16) v[e] = q8_half(w[e >> 3][(e & 7) >> 1], e & 1);
            else v[e] = (e & 1) ? q8_f32(w[e >> 3][(e & 7) >> 1] & 0xffff0000u) : q8_bf16(w[e >> 3][(e & 7) >> 1] & 0xffffu);
        }
    }
};

template <int T>
__device__ __forceinline__ void score_body(const void* __restrict__ logits, size_t ld, int vocab, const int* __restrict__ targets,
                                           float* __restrict__ logp, float* __restrict__ entropy, int top, int* __restrict__ top_idx,
                                           float* __restrict__ top_logp, int segs, int seg_len, char* __restrict__ ws, int* __restrict__ tickets) {
    __shared__ key_t_ buf[SCORE_WAVES][SCORE_CAP];
    __shared__ key_t_ best[SCORE_WAVES][SCORE_MAX_TOP];
    __shared__ float stats[SCORE_WAVES][4];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x / (unsigned)segs;
    const int seg = (int)(blockIdx.x - row * (unsigned)segs);
    const char* const z = static_cast<const char*>(logits) + row * ld * (T == Q8_F32 ? 4 : 2);
    const long long lo = (long long)seg * seg_len, hi = min(lo + seg_len, (long long)vocab);

    ScoreTop best_of{buf[wave], best[wave], top, 0, 0};
    ScoreStats st{-__builtin_inff(), 0.f, 0.f};
    float floor_v = -__builtin_inff();
    ScoreChunk<T> next;
    long long i = lo + wave * SCORE_STAGE;
    if (i < hi) next.load(z, i, hi, lane);
    for (; i < hi; i += SCORE_WAVES * SCORE_STAGE) {
        const ScoreChunk<T> cur = next;
        if (i + SCORE_WAVES * SCORE_STAGE < hi) next.load(z, i + SCORE_WAVES * SCORE_STAGE, hi, lane);
        float v[16];
        cur.get(v);
        float m = __builtin_elementwise_maximum(v[0], v[1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, v[e]), v[e + 1]);
        const float chunk_max = m;
        m = __builtin_elementwise_maximum(m, st.m);
        if (!(m == st.m)) {  // a new maximum, or NaN
            const float f = st.s > 0.f ? score_ref_diff(st.m, m) : 0.f, g = score_exp2(f);
            st.u = g > 0.f ? (st.u + st.s * f) * g : 0.f;
            st.s *= g;
            st.m = m;
        }
        // -infinity (masked, or none at all) becomes a term whose power is 0, and stays out of U
        auto term = [&](float d) {
            d = __builtin_fmaxf(d, -200.f);
            const float p = score_exp2(d);
            st.s += p;
            st.u = __builtin_fmaf(d, p, st.u);
        };
        const float mm = st.m == -__builtin_inff() ? 0.f : st.m, r = score_ref(mm);  // nothing so far: every element is -infinity
        const bool big = !(__builtin_fabsf(mm) < SCORE_BIG);
        if (__any(big)) {
#pragma unroll
            for (int e = 0; e < 16; e++) term(big ? (v[e] - mm) * 1.44269504088896341f : __builtin_fmaf(v[e], 1.44269504088896341f, -r));
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) term(__builtin_fmaf(v[e], 1.44269504088896341f, -r));
        }
        if (top > 0 && __any(!(chunk_max < floor_v))) {
            key_t_ key[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const long long at = i + ScoreChunk<T>::at(lane, e);
                key[e] = at < hi ? score_key(v[e], (unsigned)at) : 0;
            }
            best_of.take(key);
            floor_v = best_of.floor_value();
        }
    }
    auto leave = [&]() {  // this wave's results to LDS
        if (top > 0) best_of.compact();
        st = score_wave_join(st);
        if (lane == 0) {
            stats[wave][0] = st.m;
            stats[wave][1] = st.s;
            stats[wave][2] = st.u;
        }
        __syncthreads();
    };
    // wave 0: the waves' results as one; the keys of rank `lane` in the returned value
    auto join = [&]() -> key_t_ {
        st = {stats[0][0], stats[0][1], stats[0][2]};
#pragma unroll
        for (int w = 1; w < SCORE_WAVES; w++) st = score_join(st, ScoreStats{stats[w][0], stats[w][1], stats[w][2]});
        if (top == 0) return 0;
        const key_t_* const all = best[0];
        key_t_ mine[2];
        int rank[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; h++) mine[h] = all[h * 64 + lane];
        for (int e = 0; e < SCORE_WAVES * SCORE_MAX_TOP; e++) {
            const key_t_ other = all[e];
#pragma unroll
            for (int h = 0; h < 2; h++) rank[h] += other > mine[h];
        }
        score_wave_sync();
        key_t_* const o = buf[0];
        if (lane < SCORE_MAX_TOP) o[lane] = 0;
        score_wave_sync();
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (mine[h] != 0 && rank[h] < top) o[rank[h]] = mine[h];
        score_wave_sync();
        return lane < top ? o[lane] : 0;
    };
    leave();
    key_t_ ranked = 0;
    if (segs > 1) {
        // Record to the workspace by device-scope stores; complete before the ticket is drawn.  The block that draws the last
        // ticket reads all records of its row by device-scope loads.
        if (wave == 0) {
            ranked = join();
            char* const rec = ws + ((size_t)blockIdx.x) * SCORE_RECORD;
            if (lane < SCORE_MAX_TOP) __hip_atomic_store(reinterpret_cast<key_t_*>(rec + 16) + lane, ranked, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane < 3)
                __hip_atomic_store(reinterpret_cast<float*>(rec) + lane, lane == 0 ? st.m : lane == 1 ? st.s : st.u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (lane == 0) last_one = __hip_atomic_fetch_add(tickets + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs - 1;
        }
        __syncthreads();
        if (!last_one) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        if (threadIdx.x == 0) __hip_atomic_store(tickets + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
        const char* const recs = ws + row * (size_t)segs * SCORE_RECORD;
        st = {-__builtin_inff(), 0.f, 0.f};
        for (int s = threadIdx.x; s < segs; s += SCORE_WAVES * 64) {
            const float* const f = reinterpret_cast<const float*>(recs + (size_t)s * SCORE_RECORD);
            float x[3];
#pragma unroll
            for (int j = 0; j < 3; j++) x[j] = __hip_atomic_load(f + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            st = score_join(st, ScoreStats{x[0], x[1], x[2]});
        }
        best_of.count = 0;
        best_of.low = 0;
        const int total = top > 0 ? segs * SCORE_MAX_TOP : 0;
        for (int p = wave * SCORE_STAGE; p < total; p += SCORE_WAVES * SCORE_STAGE) {
            key_t_ key[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int at = p + e * 64 + lane;
                key[e] = at < total ? __hip_atomic_load(reinterpret_cast<const key_t_*>(recs + (size_t)(at / SCORE_MAX_TOP) * SCORE_RECORD + 16) + at % SCORE_MAX_TOP,
                                                        __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                                    : 0;
            }
            best_of.take(key);
        }
        leave();
    }
    if (wave != 0) return;
    ranked = join();
    const bool none = st.m == -__builtin_inff(), bad = !(st.m < __builtin_inff());
    const float log_s = __builtin_amdgcn_logf(st.s), r = score_ref(st.m);  // base 2
    auto log_p = [&](float v) {
        if (bad) return __builtin_nanf("");
        if (none) return -__builtin_inff();
        if (!(__builtin_fabsf(v) < SCORE_BIG) || !(__builtin_fabsf(st.m) < SCORE_BIG)) return (v - st.m) - log_s * 0.693147180559945309f;
        return (__builtin_fmaf(v, 1.44269504088896341f, -r) - log_s) * 0.693147180559945309f;
    };
    if (lane == 0) {
        if (entropy) entropy[row] = bad ? __builtin_nanf("") : none ? 0.f : __builtin_fmaxf((log_s - st.u / st.s) * 0.693147180559945309f, 0.f);
        if (logp) {
            const int target = targets[row];
            logp[row] = target < 0 ? 0.f : target >= vocab ? __builtin_nanf("") : log_p(q8_load1<T>(z, (size_t)target));
        }
    }
    if (lane < top) {
        if (top_idx) top_idx[row * top + lane] = (int)score_index(ranked);
        if (top_logp) top_logp[row * top + lane] = log_p(score_value(ranked));
    }
}

#define SCORE_KERNEL(NAME, T)                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void NAME(const void* logits, size_t ld, int vocab, const int* targets, float* logp,       \
                                                           float* entropy, int top, int* top_idx, float* top_logp, int segs, int seg_len,  \
                                                           char* ws, int* tickets) {                                                       \
        score_body<T>(logits, ld, vocab, targets, logp, entropy, top, top_idx, top_logp, segs, seg_len, ws, tickets);                      \
    }
SCORE_KERNEL(w4a16_token_logprobs_f32, Q8_F32)
SCORE_KERNEL(w4a16_token_logprobs_f16, Q8_F16)
SCORE_KERNEL(w4a16_token_logprobs_bf16, Q8_BF16)
