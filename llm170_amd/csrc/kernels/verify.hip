// Verification of drafted tokens against the target's distributions, from given random numbers.  A sequence has rows row0[b] .. row0[b + 1] - 1 of target logits: row i judges
// drafted token i, the last one is what follows when all are accepted.  With p, q the softmax of target and draft logits over the temperature, token x of row i is
// accepted while u_i q(x) < p(x); behind the last accepted one a token is drawn from max(0, p - q) at the first row that is not, from p at the last row: the first whose
// running sum exceeds u_last times the whole sum.  Temperature 0: accepted is the most likely token, which also follows.
//
// Two launches.  Rows: a segment of a target's or a draft's row to a workgroup, with a running maximum in each thread; it leaves (sum, maximum) of its segment, and the last
// of a row joins them and judges the row's token.  A decision wants its sum to some 10^-7, so powers are of 32 bits here, some 7 instructions an element, and the stream of the logits
// takes most of the time: 193 rows of 131072 bf16 with 129 drafts' 22.4 us (84 MB, 3.8 TB/s), 400 of 100003 f16 with 200 drafts' 31.9 (120 MB).
// Pick: of the first row that is not accepted alone, a stage of 64 lanes to a wave.  Running sums over a vocabulary meet a border between two tokens about once in V / (relative error)
// draws, so powers and sums are of 64 bits: 2^x by a polynomial of degree 8 (interpolation at Chebyshev nodes of [-1/2, 1/2], off by 1.1e-12), some 17 instructions of four
// cycles, which are what takes the time where there are many sequences: 64 of them 20.6 us (7 of arithmetic; launch, loads that depend on each other and the last workgroup's work the rest), 200 45.5 (28).
// A wave leaves sum p, sum q and, by the first launch's sums (`rough` of the draft's power is one of the target's), sum max(0, p - q) and the sum of q where p is above q: what is
// known of the whole sums then changes it by their difference times the last.  Tokens that the first launch's 10^-7 puts on the wrong side have no more than that share of themselves to
// give; where that is over 10^-9 of the whole, target and draft being nearly alike, the sums are made again with what is known now.  The last workgroup of a sequence finds the
// wave's stage that holds the draw, and the thread in it whose few neighbours do.
#include "score_common.hpp"

#define VERIFY_WAVES 4

typedef unsigned long long bits_t;

struct VerifyRow {  // what is known of a row: sum 0 where it has no distribution
    double s, sd;
    float m, md;
    int best, accepted;
};
struct VerifySum {  // of a segment: sum of powers relative to its maximum; or the key of its largest element
    double s;
    float m;
    int pad;
};
struct VerifyPart {  // of a wave's stage of a row that is drawn from: sums of the powers of target and draft; of max(0, target - rough draft); of the draft's where that is above 0, and where it is
    double v[5];     // nearly 0 (the last two of 32 bits)
};
#define VERIFY_E 0
#define VERIFY_D 1
#define VERIFY_MORE 2
#define VERIFY_D_OVER 3
#define VERIFY_D_NEAR 4
#define VERIFY_NEAR 1e-6

// 2^x, x <= 0; a NaN counts as far below
__device__ __forceinline__ double verify_exp2(double x) {
    x = __builtin_fmax(x, -1100.0);
    const double n = __builtin_rint(x), f = x - n;
    double p = 1.3255224878668817e-06;
    p = __builtin_fma(p, f, 1.5310079402249296e-05);
    p = __builtin_fma(p, f, 0.00015403455852453838);
    p = __builtin_fma(p, f, 0.0013333450568000645);
    p = __builtin_fma(p, f, 0.009618129159402558);
    p = __builtin_fma(p, f, 0.05550410941205933);
    p = __builtin_fma(p, f, 0.2402265069581299);
    p = __builtin_fma(p, f, 0.6931471805459335);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// the power of logit v relative to the maximum m; c = log2 e / temperature
__device__ __forceinline__ double verify_power(float v, float m, double c) { return verify_exp2(((double)v - (double)m) * c); }
// a segment's sum relative to the maximum of its row
__device__ __forceinline__ double verify_share(VerifySum a, float m, double c) { return a.s > 0.0 ? a.s * verify_power(a.m, m, c) : 0.0; }

__device__ __forceinline__ double verify_factor(float temp) { return 1.4426950408889634074 / (double)temp; }

__device__ __forceinline__ double verify_wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ double verify_wave_scan(double v) {  // of this lane and all below
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

__device__ __forceinline__ double verify_of_lane(double v, int lane) {
    const bits_t b = __builtin_bit_cast(bits_t, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (bits_t)hi << 32 | lo);
}

__device__ __forceinline__ void verify_put(VerifySum* p, VerifySum v) {  // device scope: past this XCD's L2
    bits_t* const b = reinterpret_cast<bits_t*>(p);
    __hip_atomic_store(b, __builtin_bit_cast(bits_t, v.s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(b + 1, (bits_t)__builtin_bit_cast(unsigned, v.m), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ VerifySum verify_get(const VerifySum* p) {
    const bits_t* const b = reinterpret_cast<const bits_t*>(p);
    const bits_t s = __hip_atomic_load(b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), m = __hip_atomic_load(b + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return {__builtin_bit_cast(double, s), q8_f32((unsigned)m), 0};
}

template <int T>
__device__ __forceinline__ void verify_rows_body(const void* __restrict__ logits, size_t ld, const void* __restrict__ draft, size_t ldd, int vocab, int t, int row_first,
                                                 const int* __restrict__ row0, int seqs, const int* __restrict__ drafted, const float* __restrict__ u,
                                                 const float* __restrict__ temps, int segs, int seg_len, VerifySum* __restrict__ sums, VerifyRow* __restrict__ rows,
                                                 int* __restrict__ tickets) {
    __shared__ double red[VERIFY_WAVES];
    __shared__ float redm[VERIFY_WAVES];
    __shared__ int counts[VERIFY_WAVES];
    __shared__ int last_one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned streams = draft ? 2 : 1, per_row = (unsigned)segs * streams;
    const int row = row_first + (int)(blockIdx.x / per_row);
    const unsigned in_row = blockIdx.x % per_row;
    const bool of_draft = in_row >= (unsigned)segs;
    const int seg = (int)(of_draft ? in_row - segs : in_row);
    constexpr int SIZE = ScoreChunk<T>::SIZE, E = ScoreChunk<T>::E;
    constexpr unsigned STAGE = ScoreChunk<T>::STAGE, STEP = VERIFY_WAVES * STAGE;
    const char* const z = static_cast<const char*>(of_draft ? draft : logits) + (size_t)row * (of_draft ? ldd : ld) * SIZE;
    const unsigned lo = (unsigned)seg * (unsigned)seg_len, hi = min(lo + (unsigned)seg_len, (unsigned)vocab);
    unsigned i = lo + wave * STAGE;
    ScoreChunk<T> next;  // asked for ahead of what the row is
    auto load = [&]() { next.load(z + (size_t)i * SIZE, hi > i ? hi - i : 0u, lane); };
    load();
    // The starts at or below the row, `below` of them: 256 probes at a time
    int below = 0;
    for (int n = seqs, step;; ) {
        step = (n + 255) >> 8;
        const int at = (int)threadIdx.x * step;
        const int here = __popcll(__ballot(at < n && row0[below + min(at, n - 1)] <= row));
        __syncthreads();
        if (lane == 0) counts[wave] = here;
        __syncthreads();
        const int c = counts[0] + counts[1] + counts[2] + counts[3];
        if (c == 0) return;  // ahead of the first sequence
        below += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (step == 1) break;
    }
    below++;
    const int end = min(row0[below], t);
    if (row >= end) return;  // behind the last sequence
    const bool last = row == end - 1;
    const float temp = temps ? temps[below - 1] : 1.f;
    const bool greedy = !(temp > 0.f), both = draft && !last && !greedy;
    if (of_draft && !both) return;
    // The factor as a 32-bit number, here for all of the row: decisions are those of a temperature 2^-25 off at most.  Never 0, which would make a number of -infinity's power.
    const float factor = greedy ? 0.f : (float)__builtin_fmin(__builtin_fmax(verify_factor(temp), 1e-30), 1e37);
    const double c = factor;

    VerifySum mine = {0.0, -__builtin_inff(), 0};
    unsigned best = 0;
    for (;; i += STEP) {
        const ScoreChunk<T> cur = next;
        const unsigned here = i;
        if (i + STEP < hi) next.load(z + (size_t)(i + STEP) * SIZE, hi - i - STEP, lane);
        float most, least;
        cur.extremes(most, least);
        if (greedy) {
            if (!(most <= mine.m)) {  // later elements of equal size come later; a NaN stays
                mine.m = __builtin_elementwise_maximum(most, mine.m);
                unsigned at = 0;
#pragma unroll
                for (int e = E - 1; e >= 0; e--)
                    if (cur.value(e) == most) at = here + ScoreChunk<T>::at(lane, e);
                best = at;
            }
        } else {
            const float m = __builtin_elementwise_maximum(most, mine.m);
            if (!(m == mine.m)) {
                mine.s = mine.s > 0.0 ? mine.s * verify_power(mine.m, m, c) : 0.0;
                mine.m = m;
            }
            const float mm = mine.m == -__builtin_inff() ? 0.f : mine.m;  // nothing so far: every element is -infinity
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    p[k] = __builtin_amdgcn_exp2f(cur.minus(e + k, mm) * factor);
                }
                mine.s += (double)((p[0] + p[1]) + (p[2] + p[3]));
            }
        }
        if (i + STEP >= hi) break;
    }
    // the workgroup's sum; or the key of its largest, the lower index of equal ones
    if (greedy) {
        bits_t key = (bits_t)score_order(mine.m) << 32 | (0xffffffffu - best);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) key = max(key, (bits_t)__shfl_xor((unsigned long long)key, d));
        if (lane == 0) red[wave] = __builtin_bit_cast(double, key);
    } else {
        const float m = score_wave_max(mine.m);
        const double s = verify_wave_sum(verify_share(mine, m, c));
        if (lane == 0) {
            red[wave] = s;
            redm[wave] = m;
        }
    }
    __syncthreads();
    VerifySum* const of_row = sums + (size_t)row * per_row;
    if (threadIdx.x == 0) {
        VerifySum all = {red[0], redm[0], 0};
        if (greedy) {
            bits_t key = __builtin_bit_cast(bits_t, red[0]);
            for (int w = 1; w < VERIFY_WAVES; w++) key = max(key, __builtin_bit_cast(bits_t, red[w]));
            all = {__builtin_bit_cast(double, key), 0.f, 0};
        } else {
            for (int w = 1; w < VERIFY_WAVES; w++) all.m = __builtin_elementwise_maximum(all.m, redm[w]);
            all.s = 0.0;
            for (int w = 0; w < VERIFY_WAVES; w++) all.s += verify_share({red[w], redm[w], 0}, all.m, c);
        }
        verify_put(of_row + in_row, all);
        // complete before the ticket is drawn; read behind the barrier that follows its return
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        last_one = __hip_atomic_fetch_add(tickets + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs * (both ? 2 : 1) - 1;
    }
    __syncthreads();
    if (!last_one) return;
    if (threadIdx.x == 0) __hip_atomic_store(tickets + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    if (wave != 0) return;
    VerifyRow r = {0.0, 0.0, 0.f, 0.f, 0, 0};
    const int x = last ? -1 : drafted[row];
    const bool there = x >= 0 && x < vocab;
    if (greedy) {
        bits_t key = 0;
        for (int s = lane; s < segs; s += 64) key = max(key, __builtin_bit_cast(bits_t, verify_get(of_row + s).s));
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) key = max(key, (bits_t)__shfl_xor((unsigned long long)key, d));
        const unsigned order = (unsigned)(key >> 32);
        r.best = (int)(0xffffffffu - (unsigned)key);
        r.s = order > score_order(-__builtin_inff()) && order < score_order(__builtin_inff()) ? 1.0 : 0.0;
        r.accepted = r.s > 0.0 && there && x == r.best;
    } else {
        auto join = [&](const VerifySum* of, float& m, double& s) {
            VerifySum a = {0.0, -__builtin_inff(), 0};
            for (int k = lane; k < segs; k += 64) {
                const VerifySum v = verify_get(of + k);
                const float both_m = __builtin_elementwise_maximum(a.m, v.m);
                a.s = verify_share(a, both_m, c) + verify_share(v, both_m, c);
                a.m = both_m;
            }
            m = score_wave_max(a.m);
            s = verify_wave_sum(verify_share(a, m, c));
            if (!(__builtin_fabsf(m) < __builtin_inff())) s = 0.0;  // nothing, infinity or NaN
        };
        join(of_row, r.m, r.s);
        if (both) join(of_row + segs, r.md, r.sd);
        if (there && r.s > 0.0) {
            const double p = verify_power(q8_load1<T>(static_cast<const char*>(logits) + (size_t)row * ld * SIZE, (size_t)x), r.m, c) / r.s;
            double q = 1.0;
            if (both && r.sd > 0.0) q = verify_power(q8_load1<T>(static_cast<const char*>(draft) + (size_t)row * ldd * SIZE, (size_t)x), r.md, c) / r.sd;
            r.accepted = (!both || r.sd > 0.0) && (double)u[row] * q < p;
        }
    }
    if (lane == 0) rows[row] = r;
}

// The first of 256 values, one per thread, whose running sum from `before` on exceeds `aim`; else (`none`) the last one above zero; else -1.  `before` becomes the sum ahead of the first
// kind; of every value it is in `starts`, and the waves' sums are in `red`.  All threads get the same.
__device__ __forceinline__ int verify_find(double v, double aim, double& before, double* red, int* found, double* starts, bool& none) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double run = verify_wave_scan(v);
    __syncthreads();
    if (lane == 63) red[wave] = run;
    if (threadIdx.x < 2) found[threadIdx.x] = threadIdx.x == 0 ? 256 : -1;
    __syncthreads();
    double ahead = before;
    for (int w = 0; w < wave; w++) ahead += red[w];
    const bool over = ahead + run > aim && v > 0.0;
    const unsigned long long those = __ballot(over), some = __ballot(v > 0.0);
    if (lane == 0) {
        if (those) atomicMin(&found[0], wave * 64 + __builtin_ctzll(those));
        if (some) atomicMax(&found[1], wave * 64 + 63 - __builtin_clzll(some));
    }
    starts[threadIdx.x] = ahead + (run - v);
    __syncthreads();
    none = found[0] == 256;
    const int at = none ? found[1] : found[0];
    if (!none) before = starts[at];
    return at;
}

template <int T>
__device__ __forceinline__ void verify_pick_body(const void* __restrict__ logits, size_t ld, const void* __restrict__ draft, size_t ldd, int vocab, int t, int seq_first,
                                                 const int* __restrict__ row0, const int* drafted, const float* __restrict__ u, const float* __restrict__ temps,
                                                 int segs, const VerifyRow* __restrict__ rows, VerifyPart* __restrict__ parts, int* __restrict__ tickets,
                                                 int* tokens, int* __restrict__ accepted) {
    __shared__ double red[VERIFY_WAVES], sums[5][VERIFY_WAVES], starts[256];
    __shared__ int found[2];
    __shared__ int last_one, chosen;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = threadIdx.x;
    const int b = seq_first + (int)(blockIdx.x / (unsigned)segs), seg = (int)(blockIdx.x % (unsigned)segs);
    const int r0 = min(max(row0[b], 0), t), r1 = min(max(row0[b + 1], r0), t);
    if (r0 >= r1) {
        if (seg == 0 && tid == 0) accepted[b] = 0;
        return;
    }
    const float temp = temps ? temps[b] : 1.f, draw = u[r1 - 1];
    int stop = r1 - 1;
    VerifyRow r;
    for (int from = r0;; from += 64) {  // what is known of 64 rows, one to a lane
        const VerifyRow mine = rows[min(from + lane, r1 - 1)];
        const unsigned long long no = __ballot(from + lane < r1 - 1 && mine.accepted == 0);
        if (!no && from + 64 < r1) continue;
        const int of = no ? __builtin_ctzll(no) : r1 - 1 - from;
        stop = from + of;
        r.s = verify_of_lane(mine.s, of);
        r.sd = verify_of_lane(mine.sd, of);
        r.m = q8_f32((unsigned)__builtin_amdgcn_readlane(__builtin_bit_cast(int, mine.m), of));
        r.md = q8_f32((unsigned)__builtin_amdgcn_readlane(__builtin_bit_cast(int, mine.md), of));
        r.best = __builtin_amdgcn_readlane(mine.best, of);
        break;
    }
    const bool greedy = !(temp > 0.f), last = stop == r1 - 1, both = draft && !last && r.sd > 0.0;
    int token = greedy && r.s > 0.0 ? r.best : -1;
    if (greedy || !(r.s > 0.0)) {
        if (seg != 0) return;
    } else {
        constexpr int SIZE = ScoreChunk<T>::SIZE, E = ScoreChunk<T>::E, PER = ScoreChunk<T>::PER;
        constexpr int STAGE = ScoreChunk<T>::STAGE;
        const char* const z = static_cast<const char*>(logits) + (size_t)stop * ld * SIZE;
        const char* const zd = static_cast<const char*>(draft) + (size_t)stop * ldd * SIZE;
        const double c = verify_factor(temp);
        const int x = last || draft ? -1 : drafted[stop];  // left out: the token that was certain to its draft
        const double rough = both ? r.s / r.sd : 0.0;  // p > q: e > d S / S_draft
        const int parts_n = segs * VERIFY_WAVES;
        VerifyPart* const of_seq = parts + (size_t)b * parts_n;
        auto load = [&](ScoreChunk<T>& to, const char* from, int part) {
            const int i = part * STAGE;
            to.load(from + (size_t)i * SIZE, i < vocab ? (unsigned)(vocab - i) : 0u, lane);
        };
        auto put = [&](int part, int k, double v) { __hip_atomic_store(reinterpret_cast<bits_t*>(of_seq[part].v + k), __builtin_bit_cast(bits_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        {
            const int part = seg * VERIFY_WAVES + wave;
            double sum[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
            ScoreChunk<T> v, d;
            load(v, z, part);
            if (both) {
                load(d, zd, part);
                float over = 0.f, near = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const double p = verify_power(v.value(e), r.m, c), q = verify_power(d.value(e), r.md, c), more = __builtin_fma(-q, rough, p);
                    const float qf = (float)q;
                    sum[VERIFY_E] += p;
                    sum[VERIFY_D] += q;
                    sum[VERIFY_MORE] += __builtin_fmax(more, 0.0);
                    over += more > 0.0 ? qf : 0.f;
                    near += __builtin_fabs(more) <= VERIFY_NEAR * p ? qf : 0.f;
                    // 2 powers of each under way at once: more take the registers of whole waves
                    if (e % 2 == 1) asm volatile("" : "+v"(sum[VERIFY_E]), "+v"(sum[VERIFY_D]), "+v"(sum[VERIFY_MORE]), "+v"(over), "+v"(near));
                }
                sum[VERIFY_D_OVER] = over;
                sum[VERIFY_D_NEAR] = near;
#pragma unroll
                for (int k = 0; k < 5; k++) {
                    sum[k] = verify_wave_sum(sum[k]);
                    if (lane == k) put(part, k, sum[k]);
                }
            } else {
                const int out = x - part * STAGE - ScoreChunk<T>::at(lane, 0);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const double p = verify_power(v.value(e), r.m, c);
                    sum[VERIFY_E] += out == ScoreChunk<T>::at(0, e) ? 0.0 : p;
                    if (e % 2 == 1) asm volatile("" : "+v"(sum[VERIFY_E]));
                }
                sum[VERIFY_E] = verify_wave_sum(sum[VERIFY_E]);
                if (lane == 0) put(part, VERIFY_E, sum[VERIFY_E]);
            }
        }
        // complete before the ticket is drawn; read behind the barrier that follows its return
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (segs > 1) {
            if (tid == 0) last_one = __hip_atomic_fetch_add(tickets + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == segs - 1;
            __syncthreads();
            if (!last_one) return;
            if (tid == 0) __hip_atomic_store(tickets + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
        }
        // sums over the workgroup, or the first alone; all threads get them
        auto of_all = [&](double (&v)[5], int count) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 5; k++) {
                if (k >= count) break;
                const double w = verify_wave_sum(v[k]);
                if (lane == 0) sums[k][wave] = w;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 5; k++) v[k] = k < count ? (sums[k][0] + sums[k][1]) + (sums[k][2] + sums[k][3]) : 0.0;
        };
        // Parts tid, tid + 256, ..: the first is kept in registers
        auto fetch = [&](int part, double (&v)[5]) {
#pragma unroll
            for (int k = 0; k < 5; k++) {
                v[k] = 0.0;
                if (part < parts_n && (k == 0 || both))
                    v[k] = __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const bits_t*>(of_seq[part].v + k), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            }
        };
        double first[5], all[5];
        fetch(tid, first);
#pragma unroll
        for (int k = 0; k < 5; k++) all[k] = first[k];
        for (int part = tid + 256; part < parts_n; part += 256) {
            double v[5];
            fetch(part, v);
#pragma unroll
            for (int k = 0; k < 5; k++) all[k] += v[k];
        }
        of_all(all, both ? 5 : 1);
        const double inv = 1.0 / all[VERIFY_E], inv_d = both ? 1.0 / all[VERIFY_D] : 0.0;
        const double left = both ? rough - all[VERIFY_E] * inv_d : 0.0;  // max(0, p - q) by what is known now: that of the rough factor, and this much of the draft's
        bool only_p = !both, again = false;
        auto weight = [&](float v, float d, int at) {
            const double p = verify_power(v, r.m, c) * inv;
            if (only_p) return at == x ? 0.0 : p;
            return __builtin_fmax(p - verify_power(d, r.md, c) * inv_d, 0.0);
        };
        auto share = [&](const double (&v)[5]) {
            return only_p ? v[VERIFY_E] * inv : again ? v[VERIFY_MORE] : __builtin_fma(left, v[VERIFY_D_OVER], v[VERIFY_MORE]) * inv;  // below 0 where tokens are nearly alike
        };
        double whole = only_p ? (all[VERIFY_E] > 0.0 ? 1.0 : 0.0) : share(all);
        if (both) {
            const double off = __builtin_fabs(rough * all[VERIFY_D] * inv - 1.0);
            again = !(off < VERIFY_NEAR) || off * rough * all[VERIFY_D_NEAR] * inv > 1e-9 * whole;
            if (again) {
                for (int part = wave; part < parts_n; part += VERIFY_WAVES) {
                    ScoreChunk<T> v, d;
                    load(v, z, part);
                    load(d, zd, part);
                    double w = 0.0;
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        w += weight(v.value(e), d.value(e), -1);
                        if (e % 2 == 1) asm volatile("" : "+v"(w));
                    }
                    w = verify_wave_sum(w);
                    if (lane == 0) put(part, VERIFY_MORE, w);
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                fetch(tid, first);
                double v[5] = {first[VERIFY_MORE], 0.0, 0.0, 0.0, 0.0};
                for (int part = tid + 256; part < parts_n; part += 256) {
                    double w[5];
                    fetch(part, w);
                    v[0] += w[VERIFY_MORE];
                }
                of_all(v, 1);
                whole = v[0];
            }
        }
        // Of a part, thread i has the PER neighbours from i PER on: their weights, and the sum of them
        double weights[PER];
        auto of_run = [&](int part) {
            const int from = part * STAGE + tid * PER;
            ScoreChunk<T> v, d;
            if (from + PER <= vocab) {
                v.w[0] = *reinterpret_cast<const u4_any_t*>(z + (size_t)from * SIZE);
                if (!only_p) d.w[0] = *reinterpret_cast<const u4_any_t*>(zd + (size_t)from * SIZE);
#pragma unroll
                for (int e = 0; e < PER; e++) weights[e] = weight(v.value(e), only_p ? 0.f : d.value(e), from + e);
            } else {
#pragma unroll
                for (int e = 0; e < PER; e++) weights[e] = from + e < vocab ? weight(q8_load1<T>(z, (size_t)(from + e)), only_p ? 0.f : q8_load1<T>(zd, (size_t)(from + e)), from + e) : 0.0;
            }
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < PER; e++) sum += weights[e];
            return sum;
        };
        // Drawn from p where p is nowhere above q, or where no token of the segment that the draw falls into is left at the second look
        for (int attempt = 0; attempt < 2 && token < 0; attempt++) {
            if (attempt == 1) {
                if (only_p) break;
                only_p = true;
                whole = 1.0;
            }
            if (!(whole > 0.0)) continue;
            const double aim = (double)draw * whole;
            double before = 0.0, from = 0.0;
            int at = -1;
            bool none = true;
            for (int part = 0; part < parts_n && none; part += 256) {
                double ahead = from, v[5];
                if (part > 0) fetch(part + tid, v);
                const int f = verify_find(part > 0 ? share(v) : share(first), aim, ahead, red, found, starts, none);
                if (f >= 0) {
                    at = part + f;
                    before = none ? starts[f] : ahead;
                }
                from += red[0] + red[1] + red[2] + red[3];
            }
            if (at < 0) continue;
            if (tid == 0) chosen = -1;
            const int f = verify_find(of_run(at), aim, before, red, found, starts, none);
            if (tid == f) {
                double run = starts[f];
                int over = -1, some = -1;
#pragma unroll
                for (int e = 0; e < PER; e++) {
                    run += weights[e];
                    some = weights[e] > 0.0 ? e : some;
                    over = over < 0 && weights[e] > 0.0 && run > aim ? e : over;
                }
                if (some >= 0) chosen = at * STAGE + f * PER + (over >= 0 ? over : some);
            }
            __syncthreads();
            token = chosen;
        }
        if (token < 0) token = x;  // all of p is on the token that was left out
    }
    for (int i = r0 + tid; i < r1; i += 256) tokens[i] = i < stop ? drafted[i] : i == stop ? token : -1;
    if (tid == 0) accepted[b] = stop - r0;
}

#define VERIFY_KERNELS(NAME, T)                                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void w4a16_verify_rows_##NAME(                                                    \
        const void* logits, size_t ld, const void* draft, size_t ldd, int vocab, int t, int row_first, const int* row0, int seqs, const int* drafted, \
        const float* u, const float* temps, int segs, int seg_len, VerifySum* sums, VerifyRow* rows, int* tickets) {               \
        verify_rows_body<T>(logits, ld, draft, ldd, vocab, t, row_first, row0, seqs, drafted, u, temps, segs, seg_len, sums, rows, tickets); \
    }                                                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void w4a16_verify_pick_##NAME(                                                    \
        const void* logits, size_t ld, const void* draft, size_t ldd, int vocab, int t, int seq_first, const int* row0, const int* drafted, const float* u, \
        const float* temps, int segs, const VerifyRow* rows, VerifyPart* parts, int* tickets, int* tokens, int* accepted) {  \
        verify_pick_body<T>(logits, ld, draft, ldd, vocab, t, seq_first, row0, drafted, u, temps, segs, rows, parts, tickets, tokens, accepted); \
    }
VERIFY_KERNELS(f32, Q8_F32)
VERIFY_KERNELS(f16, Q8_F16)
VERIFY_KERNELS(bf16, Q8_BF16)
