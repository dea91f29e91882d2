// Scoring of rows of logits z[V]: the log probability of a given token, the entropy of the distribution, and the most likely
// tokens with theirs.  One pass over the row with a running maximum:
//   S = sum 2^(z L - r),  U = sum (z L - r) 2^(z L - r),  L = log2 e, r = fl(max z * L), each term one fused multiply-add;
//   log p_j = ln 2 * ((z_j L - r) - log2 S),  entropy = ln 2 * (log2 S - U / S).
// r is the same rounded number in every term: what its rounding (half a last place of m L, m the largest z so far) puts on an exponent is on all
// of them, and cancels.  That holds while it is far below one; from |m| = 2^20 on (2^-4 there; 128 and more from 2^31 on, where the largest power
// leaves f32) the difference is taken before the factor, (z - m) L, and where z L itself could leave f32 (beyond 1e38: the lowest value of a type as a
// mask) the exponent is held at -200.  Lanes of either kind meet where finite masks leave some lanes nothing else: a joining needs the distance of
// their references, which one fused multiply-add gives.  A row that holds NaN or +infinity has NaN for all its
// numbers; a row of -infinity alone gives its tokens -infinity and the entropy 0.
//
// The best tokens: an element is the key (order-preserving image of its value << 32 | ~index), so that no two are alike and equal
// values rank by index.  Every wave keeps a list of candidates in LDS.  What a candidate has to reach: with k' = top_k / (waves at
// work), rounded up, the smallest over the waves of the k'-th largest of a wave's 64 lane maxima so far; top_k elements are known to be as
// large (top_k <= 4: k' = top_k, and the largest over the waves).  It leaves few more than top_k elements of the first stage, and ever fewer later.  Only lanes whose maximum or 32
// reaches it are looked at: they put their elements down in LDS and the wave goes over them 64 at a time.  A list grown too long is
// cut to its best, whose last key is what the wave's later elements have to exceed: that bounds it where many values are equal, too.
// A workgroup runs through little of this more than a few times, so that the code's way from memory is most of a short launch: every
// part of it is there once.
// A row goes to one workgroup or, where there are few rows, to several: each leaves its record in the workspace and draws a
// ticket, the last one joins them.
// Launches back to back: 2048 x 100003 f16 with its best token 90 us, 4.6 TB/s: the exponentials' issue and the stream, which a copy runs at 5.1
// TB/s.  64 x 131072 bf16, 20 best, 20.7 us, without alternatives 12.5; 1 x 32000 f32, 5 best, 9.9, without 5.4: chains of latencies, not bytes: one
// stage for every wave, the ranking of its candidates, the joining of the waves and of the records.  64 x 131072 with 99.9 % ruled out 36.5 us: where a
// stage holds nothing else, all lanes of -infinity reach the bound.
#include "q8_common.hpp"

#define SCORE_MAX_TOP 32
#define SCORE_STAGE_BYTES 4096  // of a wave's stage, 64 per lane
#define SCORE_WAVES 4
#define SCORE_LIST 128         // places of a wave's list: 2 SCORE_MAX_TOP carried over and 64 of one step
#define SCORE_BATCH 32         // lanes that put their elements down at a time, half as many where they have 32
#define SCORE_RECORD 272       // bytes of a workgroup's record: max, S, U, padding, SCORE_MAX_TOP keys

typedef unsigned long long key_t_;

struct ScoreStats {
    float m, s, u;  // largest logit, S and U relative to score_ref(m)
};

#define SCORE_LOG2E 1.44269504088896341f
#define SCORE_BIG 1048576.0f  // maxima from here on are taken off before the factor
#define SCORE_FAR 1e38f       // their product with the factor could leave f32
// A term of z is 2^((z - c) L - r); one of c and r is 0.  NaN and the infinities count as big; no f16 (T) does, rows of those have NaN anyhow
// (2048 x 100003 f16 with this test in it 96.5 us, without 92).
struct ScoreRef {
    float c, r;
};
template <int T>
__device__ __forceinline__ ScoreRef score_ref(float m) {
    const bool big = T != Q8_F16 && !(__builtin_fabsf(m) < SCORE_BIG);
    return {big ? m : 0.f, big ? 0.f : m * SCORE_LOG2E};
}
// What the powers relative to a's reference are multiplied with, as an exponent, to be relative to b's; a <= b
template <int T>
__device__ __forceinline__ float score_ref_diff(float a, float b) {
    const ScoreRef ra = score_ref<T>(a), rb = score_ref<T>(b);
    const float d = T == Q8_F16 ? ra.r - rb.r : __builtin_fmaf(ra.c - rb.c, SCORE_LOG2E, ra.r - rb.r);
    return a == b ? 0.f : __builtin_fmaxf(d, -1e30f);
}
__device__ __forceinline__ float score_exp2(float d) { return __builtin_amdgcn_exp2f(d); }

// Sums relative to one maximum, re-expressed relative to a larger one and added.  -infinity: nothing there yet.
template <int T>
__device__ __forceinline__ ScoreStats score_join(ScoreStats a, ScoreStats b) {
    ScoreStats o;
    o.m = __builtin_elementwise_maximum(a.m, b.m);  // a NaN stays
    const float da = a.s > 0.f ? score_ref_diff<T>(a.m, o.m) : 0.f, db = b.s > 0.f ? score_ref_diff<T>(b.m, o.m) : 0.f;
    const float fa = score_exp2(da), fb = score_exp2(db);
    o.s = a.s * fa + b.s * fb;
    const float ua = a.u + a.s * da, ub = b.u + b.s * db;
    o.u = (fa > 0.f ? ua * fa : 0.f) + (fb > 0.f ? ub * fb : 0.f);
    return o;
}

// Lane 63 of the result combines all 64: rows of 16 by shifts, then across the rows
template <int CTRL, int ROWS>
__device__ __forceinline__ float score_dpp(float old, float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float score_wave_sum(float v) {
    v += score_dpp<0x111, 0xf>(0.f, v);
    v += score_dpp<0x112, 0xf>(0.f, v);
    v += score_dpp<0x114, 0xf>(0.f, v);
    v += score_dpp<0x118, 0xf>(0.f, v);
    v += score_dpp<0x142, 0xa>(0.f, v);
    v += score_dpp<0x143, 0xc>(0.f, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float score_wave_max(float v) {  // NaN where a lane has one
    v = __builtin_elementwise_maximum(v, score_dpp<0x111, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x112, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x114, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x118, 0xf>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x142, 0xa>(v, v));
    v = __builtin_elementwise_maximum(v, score_dpp<0x143, 0xc>(v, v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
template <int T>
__device__ __forceinline__ ScoreStats score_wave_join(ScoreStats a) {
    ScoreStats o;
    o.m = score_wave_max(a.m);
    const float d = a.s > 0.f ? score_ref_diff<T>(a.m, o.m) : 0.f, f = score_exp2(d);
    o.s = score_wave_sum(a.s * f);
    o.u = score_wave_sum(f > 0.f ? (a.u + a.s * d) * f : 0.f);
    return o;
}

// Larger for the larger value; NaN above all, -0 as 0
__device__ __forceinline__ unsigned score_order(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);
    return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ key_t_ score_key(float v, unsigned index) { return (key_t_)score_order(v) << 32 | (0xffffffffu - index); }
__device__ __forceinline__ float score_value(key_t_ k) {
    const unsigned o = (unsigned)(k >> 32);
    return __builtin_bit_cast(float, (o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned score_index(key_t_ k) { return 0xffffffffu - (unsigned)k; }

__device__ __forceinline__ key_t_ score_lane(key_t_ v, int lane) {
    return (key_t_)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ void score_wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The candidates of one wave; uniform for the wave.
struct ScoreTop {
    key_t_* list;  // LDS, SCORE_LIST + 4
    int top, count;
    key_t_ low;    // an element has to exceed it; 0 is below every key

    // one more key per lane where `in`
    __device__ __forceinline__ void step(key_t_ key, bool in) {
        const int lane = threadIdx.x & 63;
        const unsigned long long all = __ballot(in);
        if (in) list[count + __builtin_amdgcn_mbcnt_hi((unsigned)(all >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)all, 0))] = key;
        count += __popcll(all);
        // Room beyond `top`, or the last of the first stage's keys would cost a cut each: 2538 rows of 1249 f16, top 32, 49 us, with room 29
        if (count <= max(SCORE_MAX_TOP, 2 * top)) return;
        // cut to the `top` best, best first
        if (lane < 4) list[count + lane] = 0;  // the loop goes by four
        score_wave_sync();
        key_t_ mine[2];
        int rank[2] = {0, 0};
        mine[0] = lane < count ? list[lane] : 0;
        mine[1] = 64 + lane < count ? list[64 + lane] : 0;
#pragma unroll 1
        for (int e = 0; e < count; e += 4) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const key_t_ other = list[e + j];
                rank[0] += other > mine[0];
                rank[1] += other > mine[1];
            }
        }
        score_wave_sync();
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (mine[h] != 0 && rank[h] < top) list[rank[h]] = mine[h];
        score_wave_sync();
        count = min(count, top);
        if (count == top) low = max(low, score_lane(list[top - 1], 0));
    }
};

// An image that `want` lanes at least, and not many more, reach with theirs: between the largest and the smallest by halves.
__device__ __forceinline__ unsigned score_reach(float best, int want) {
    const unsigned o = score_order(best);
    unsigned hi = q8_wave_max(o), lo = ~q8_wave_max(~o);
    if (__popcll(__ballot(o >= hi)) >= want) return hi;
#pragma unroll 1
    while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        const int c = __popcll(__ballot(o >= mid));
        if (c < want) {
            hi = mid;
        } else {
            lo = mid;
            if (c <= want + want / 4) break;
        }
    }
    return lo;
}

// 64 bytes of raw elements per lane: E of them, element e is index at(e) of the stage
template <int T>
struct ScoreChunk {
    static constexpr int N = 4, PER = T == Q8_F32 ? 4 : 8, SIZE = T == Q8_F32 ? 4 : 2, E = N * PER, STAGE = 64 * E;
    u4_t w[N];

    static __device__ __forceinline__ int at(int lane, int e) { return (e / PER) * (PER * 64) + lane * PER + e % PER; }
    // p: the stage's first element (uniform), n: the elements that there are from it on; those behind them read as -infinity
    __device__ __forceinline__ void load(const char* p, unsigned n, int lane) {
        if (n >= STAGE) {
#pragma unroll
            for (int j = 0; j < N; j++) w[j] = *reinterpret_cast<const u4_any_t*>(p + lane * 16 + j * 1024);
            return;
        }
        const unsigned none = T == Q8_F32 ? 0xff800000u : T == Q8_F16 ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int j = 0; j < N; j++) {
            w[j] = (u4_t){none, none, none, none};
            if (at(lane, j * PER) + PER <= (int)n) w[j] = *reinterpret_cast<const u4_any_t*>(p + lane * 16 + j * 1024);
        }
        // the 16 bytes of one lane that the end lies in
        const int left = (int)n % PER, vec = (int)n / PER;
        if (left == 0) return;
        if (lane == vec % 64) {
            u4_t t = {none, none, none, none};
#pragma unroll
            for (int d = 0; d < PER - 1; d++) {
                const unsigned at_d = (n - left + min(d, left - 1)) * SIZE;
                if (T == Q8_F32) {
                    const unsigned v = *reinterpret_cast<const unsigned*>(p + at_d);
                    if (d < left) t[d] = v;
                } else {
                    const unsigned v = *reinterpret_cast<const uint16_t*>(p + at_d);
                    if (d < left) t[d / 2] = d & 1 ? (t[d / 2] & 0xffffu) | v << 16 : (t[d / 2] & 0xffff0000u) | v;
                }
            }
#pragma unroll
            for (int j = 0; j < N; j++)
                if (j == vec / 64) w[j] = t;
        }
    }
    // Forgets the values that were computed from the raw elements, which else stay in registers from one use to the next
    __device__ __forceinline__ void fresh() {
#pragma unroll
        for (int i = 0; i < N * 4; i++) {
            unsigned d = w[i / 4][i % 4];
            asm volatile("" : "+v"(d));
            w[i / 4][i % 4] = d;
        }
    }
    __device__ __forceinline__ float value(int e) const {
        const unsigned d = w[e / PER][T == Q8_F32 ? e % PER : e % PER / 2];
        if (T == Q8_F32) return q8_f32(d);
        if (T == Q8_F16) return q8_half(d, e & 1);
        return (e & 1) ? q8_f32(d & 0xffff0000u) : q8_bf16(d & 0xffffu);
    }
    // value(e) * L - r, one rounding; an f16 enters the multiply-add as it is
    __device__ __forceinline__ float scaled(int e, float r) const {
        if (T != Q8_F16) return __builtin_fmaf(value(e), SCORE_LOG2E, -r);
        float d;
        const unsigned h = w[e / PER][e % PER / 2];
        const float l = SCORE_LOG2E;
        if (e & 1) asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "s"(l), "v"(r));
        else asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "s"(l), "v"(r));
        return d;
    }
    // the largest and the smallest (NaN if there is one); f16 two at a time
    __device__ __forceinline__ void extremes(float& most, float& least) const {
        if (T == Q8_F16) {
            auto pair = [&](int i) { const unsigned d = w[i / 4][i % 4]; return __builtin_bit_cast(h2_t, d); };
            h2_t a = pair(0), b = pair(0);
#pragma unroll
            for (int i = 1; i < E / 2; i++) {
                a = __builtin_elementwise_maximum(a, pair(i));
                b = __builtin_elementwise_minimum(b, pair(i));
            }
            most = __builtin_elementwise_maximum((float)a[0], (float)a[1]);
            least = __builtin_elementwise_minimum((float)b[0], (float)b[1]);
        } else {
            most = __builtin_elementwise_maximum(value(0), value(1));
            least = __builtin_elementwise_minimum(value(0), value(1));
#pragma unroll
            for (int e = 2; e < E; e += 2) {
                most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, value(e)), value(e + 1));
                least = __builtin_elementwise_minimum(__builtin_elementwise_minimum(least, value(e)), value(e + 1));
            }
        }
    }
};

template <int T>
__device__ __forceinline__ void score_body(const void* __restrict__ logits, size_t ld, int vocab, const int* __restrict__ targets,
                                           float* __restrict__ logp, float* __restrict__ entropy, int top, int* __restrict__ top_idx,
                                           float* __restrict__ top_logp, int segs, int seg_len, char* __restrict__ ws, int* __restrict__ tickets) {
    __shared__ key_t_ lists[SCORE_WAVES][SCORE_LIST + 4];
    __shared__ key_t_ joined[SCORE_MAX_TOP];
    __shared__ float elements[SCORE_WAVES][SCORE_BATCH * 16];
    __shared__ unsigned firsts[SCORE_WAVES][SCORE_BATCH];
    __shared__ float stats[SCORE_WAVES][4];
    __shared__ int counts[SCORE_WAVES];
    __shared__ unsigned reaches[SCORE_WAVES];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x / (unsigned)segs;
    const int seg = (int)(blockIdx.x - row * (unsigned)segs);
    const char* const z = static_cast<const char*>(logits) + row * ld * (T == Q8_F32 ? 4 : 2);
    const unsigned lo = (unsigned)seg * (unsigned)seg_len, hi = min(lo + (unsigned)seg_len, (unsigned)vocab);

    // the target's logit, asked for ahead of the row: a chain of two loads
    const int target = logp ? targets[row] : -1;
    const float target_z = target >= 0 && target < vocab ? q8_load1<T>(z, (size_t)target) : __builtin_nanf("");
    constexpr int E = ScoreChunk<T>::E, BATCH = SCORE_BATCH * 16 / E;  // lanes that put their elements down at a time
    constexpr unsigned STAGE = ScoreChunk<T>::STAGE, STEP = SCORE_WAVES * STAGE;
    unsigned i = lo + wave * STAGE;
    ScoreChunk<T> next;  // a wave without elements has a stage of -infinity
    auto load = [&]() { next.load(z + (size_t)i * ScoreChunk<T>::SIZE, hi > i ? hi - i : 0u, lane); };
    load();
    // waves that have elements, and the lane maximum of each that counts
    const int at_work = (int)min((hi - lo + STAGE - 1) / STAGE, (unsigned)SCORE_WAVES), want = top <= 4 ? top : (top + at_work - 1) / at_work;
    const char* const recs = ws + row * (size_t)segs * SCORE_RECORD;

    ScoreTop best{lists[wave], top, 0, 0};
    ScoreStats st{-__builtin_inff(), 0.f, 0.f};
    key_t_ ranked = 0;  // lane l: the l-th best, in the end
    for (bool records = false, first = true;;) {  // the row's elements; then, in the last workgroup of several, the records
        ScoreChunk<T> cur;
        unsigned need = 0, mine = 0;
        bool over = false, took = false;
        if (!records) {
            cur = next;
            const unsigned here = i;
            i += STEP;
            if (i < hi) load();
            float most, least;
            cur.extremes(most, least);
            cur.fresh();
            const float m = __builtin_elementwise_maximum(most, st.m);
            if (!(m == st.m)) {  // a new maximum, or NaN
                const float f = st.s > 0.f ? score_ref_diff<T>(st.m, m) : 0.f, g = score_exp2(f);
                st.u = g > 0.f ? (st.u + st.s * f) * g : 0.f;
                st.s *= g;
                st.m = m;
            }
            float mm = st.m == -__builtin_inff() ? 0.f : st.m;  // nothing so far: every element is -infinity
            asm volatile("" : "+v"(mm));  // its product once, here: not in both ways that lead here
            const ScoreRef rel = score_ref<T>(mm);
            if (__any(rel.c != 0.f || !(least > -SCORE_FAR))) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    // -infinity (masked, or none at all) becomes a term whose power is 0, and stays out of U
                    const float d = __builtin_fmaxf(__builtin_fmaf(cur.value(e) - rel.c, SCORE_LOG2E, -rel.r), -200.f), p = score_exp2(d);
                    st.s += p;
                    st.u = __builtin_fmaf(d, p, st.u);
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // not all terms' registers at once
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float d = cur.scaled(e, rel.r), p = score_exp2(d);
                    st.s += p;
                    st.u = __builtin_fmaf(d, p, st.u);
                }
            }
            if (top > 0) {
                if (first) {
                    const unsigned t = score_reach(st.m, want);
                    if (lane == 0) reaches[wave] = t;
                    __syncthreads();
                    first = false;
                }
                unsigned least_of = 0xffffffffu, most_of = 0;
#pragma unroll
                for (int w = 0; w < SCORE_WAVES; w++) {
                    const unsigned x = __hip_atomic_load(&reaches[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    if (w < at_work) least_of = min(least_of, x), most_of = max(most_of, x);
                }
                need = top <= 4 ? most_of : least_of;
                need = (unsigned)__builtin_amdgcn_readfirstlane((int)need);
                mine = here + ScoreChunk<T>::at(lane, 0);
                const unsigned o = score_order(most), low_o = (unsigned)(best.low >> 32);
                over = mine < hi && o >= need && (o > low_o || (o == low_o && mine < score_index(best.low)));
            }
        }
        for (;;) {
            int steps, from = 0;
            if (!records) {
                const unsigned long long all = __ballot(over);
                if (all == 0) break;
                took = true;
                const int slot = __builtin_amdgcn_mbcnt_hi((unsigned)(all >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)all, 0));
                if (over && slot < BATCH) {
                    cur.fresh();
                    firsts[wave][slot] = mine;
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<f4_t*>(&elements[wave][slot * E + e]) = (f4_t){cur.value(e), cur.value(e + 1), cur.value(e + 2), cur.value(e + 3)};
                    over = false;
                }
                from = min(__popcll(all), BATCH);
                steps = (from * E + 63) >> 6;
                score_wave_sync();
            } else {
                steps = top > 0 ? (segs * SCORE_MAX_TOP - wave * 64 + 255) >> 8 : 0;  // 64 places at a time to one wave after the other
            }
#pragma unroll 1
            for (int s = 0; s < steps; s++) {
                key_t_ key = 0;
                if (!records) {
                    const int slot = s * (64 / E) + lane / E;
                    if (slot < from) {
                        const unsigned index = firsts[wave][slot] + ScoreChunk<T>::at(0, lane % E);
                        if (index < hi) key = score_key(elements[wave][s * 64 + lane], index);
                    }
                } else {
                    const int at = (s * SCORE_WAVES + wave) * 64 + lane, place = at % SCORE_MAX_TOP;
                    if (at < segs * SCORE_MAX_TOP && place < top)
                        key = __hip_atomic_load(reinterpret_cast<const key_t_*>(recs + (size_t)(at / SCORE_MAX_TOP) * SCORE_RECORD + 16) + place,
                                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                best.step(key, key > best.low && (unsigned)(key >> 32) >= need);
            }
            if (records) break;
        }
        if (!records) {
            if (i < hi) {
                if (took) {
                    const unsigned t = score_reach(st.m, want);  // any wave may read the old one meanwhile: it holds too
                    if (lane == 0) __hip_atomic_store(&reaches[wave], t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                }
                continue;
            }
        }
        // the waves' results as one: their sums in wave 0, their lists, each ranked by its own wave, in `joined`
        if (threadIdx.x < SCORE_MAX_TOP) joined[threadIdx.x] = 0;
        st = score_wave_join<T>(st);
        if (lane < 4) best.list[best.count + lane] = 0;  // the loop goes by four
        if (lane == 0) {
            stats[wave][0] = st.m;
            stats[wave][1] = st.s;
            stats[wave][2] = st.u;
            counts[wave] = best.count;
        }
        __syncthreads();
        if (top > 0) {
            const key_t_ mine = lane < best.count ? best.list[lane] : 0;
            int rank = 0;
#pragma unroll 1
            for (int w = 0; w < SCORE_WAVES; w++) {
                const int n = __builtin_amdgcn_readfirstlane(counts[w]);
#pragma unroll 1
                for (int e = 0; e < n; e += 4) {
#pragma unroll
                    for (int j = 0; j < 4; j++) rank += lists[w][e + j] > mine;
                }
            }
            if (mine != 0 && rank < top) joined[rank] = mine;
            __syncthreads();
        }
        if (wave == 0) {
            st = {stats[0][0], stats[0][1], stats[0][2]};
#pragma unroll
            for (int w = 1; w < SCORE_WAVES; w++) st = score_join<T>(st, ScoreStats{stats[w][0], stats[w][1], stats[w][2]});
            ranked = lane < top ? joined[lane] : 0;
        }
        if (records || segs == 1) break;
        // Record to the workspace by device-scope stores, complete before the ticket is drawn.  The block that draws the last ticket
        // reads all records of its row by device-scope loads, issued behind the barrier that follows the ticket's return: neither is
        // served from a cache that is not coherent, so that no cache is invalidated or written back (an acquire fence at device
        // scope stalls the XCD's L2: 4000 rows of 8000 in two segments 239 us, without it 82).
        if (wave == 0) {
            char* const rec = ws + ((size_t)blockIdx.x) * SCORE_RECORD;
            if (lane < top) __hip_atomic_store(reinterpret_cast<key_t_*>(rec + 16) + lane, ranked, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane < 3)
                __hip_atomic_store(reinterpret_cast<float*>(rec) + lane, lane == 0 ? st.m : lane == 1 ? st.s : st.u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (lane == 0) last_one = __hip_atomic_fetch_add(tickets + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs - 1;
        }
        __syncthreads();
        if (!last_one) return;
        if (threadIdx.x == 0) __hip_atomic_store(tickets + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
        st = {-__builtin_inff(), 0.f, 0.f};
        if ((int)threadIdx.x < segs) {
            const float* const f = reinterpret_cast<const float*>(recs + (size_t)threadIdx.x * SCORE_RECORD);
            st.m = __hip_atomic_load(f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            st.s = __hip_atomic_load(f + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            st.u = __hip_atomic_load(f + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        best.count = 0;
        best.low = 0;
        records = true;
    }
    if (wave != 0) return;
    const bool none = st.m == -__builtin_inff(), bad = !(st.m < __builtin_inff());
    const float log_s = __builtin_amdgcn_logf(st.s);  // base 2
    const ScoreRef rel = score_ref<T>(st.m);
    auto log_p = [&](float v) {
        if (bad) return __builtin_nanf("");
        if (none) return -__builtin_inff();
        if (!(__builtin_fabsf(v) < SCORE_FAR) || rel.c != 0.f) return (v - st.m) - log_s * 0.693147180559945309f;
        return (__builtin_fmaf(v, SCORE_LOG2E, -rel.r) - log_s) * 0.693147180559945309f;
    };
    if (lane == 0) {
        if (entropy) entropy[row] = bad ? __builtin_nanf("") : none ? 0.f : __builtin_fmaxf((log_s - st.u / st.s) * 0.693147180559945309f, 0.f);
        if (logp) logp[row] = target < 0 ? 0.f : target >= vocab ? __builtin_nanf("") : log_p(target_z);
    }
    if (lane < top) {
        if (top_idx) top_idx[row * top + lane] = (int)score_index(ranked);
        if (top_logp) top_logp[row * top + lane] = log_p(score_value(ranked));
    }
}

// The most waves per SIMD whose registers (79, 88, 111) need no spilling.  One wave more, spilled: 2048 x 50001 f32, 20 best, 124 us for 84, 2048 x
// 100003 f16, 1 best, 108 for 90, bf16 114 for 90.
#define SCORE_KERNEL(NAME, T, WAVES_PER_SIMD)                                                                                                              \
    extern "C" __global__ __launch_bounds__(256, WAVES_PER_SIMD) void NAME(const void* logits, size_t ld, int vocab, const int* targets, float* logp,       \
                                                           float* entropy, int top, int* top_idx, float* top_logp, int segs, int seg_len,  \
                                                           char* ws, int* tickets) {                                                       \
        score_body<T>(logits, ld, vocab, targets, logp, entropy, top, top_idx, top_logp, segs, seg_len, ws, tickets);                      \
    }
SCORE_KERNEL(w4a16_token_logprobs_f32, Q8_F32, 6)
SCORE_KERNEL(w4a16_token_logprobs_f16, Q8_F16, 5)
SCORE_KERNEL(w4a16_token_logprobs_bf16, Q8_BF16, 4)
