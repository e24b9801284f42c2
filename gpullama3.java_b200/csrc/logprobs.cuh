// logprobs.cuh -- log probabilities of given tokens, entropy and the most likely alternatives of logits rows, in one pass over the row.
//
// With M the largest logit and Z' = sum of exp(x - M) over every entry but ONE of the largest: log p(t) = x_t - M - log1p(Z'), H = log1p(Z') - S / (1 + Z') with
// S = sum (x - M) exp(x - M).  Leaving the largest entry out of the sum keeps the small ones that a sum starting at 1 would round away: a sure model's log p(t) = -log1p(Z').
// Sums of parts (m, z, s) join as z1 + (1 + z2) e^d, s1 + e^d (s2 + d (1 + z2)) with d = m2 - m1 <= 0.
// Alternatives go by value, equal ones by index: 64-bit keys (the value's bits, ordered as integers | ~index), no two alike.  A NaN is no alternative.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace lp {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;
typedef unsigned long long u64;

constexpr int THREADS = 256, PER_THREAD = 16, BATCH = THREADS * PER_THREAD, MAX_TOP = 32, MAX_CLUSTER = 8; // (clusters of 16 start late: 37 rows took 21 us with them, 12 with 8)
constexpr int PUSHERS = 64;                                // threads that may add candidates in a batch: more of them raise the threshold first
constexpr int MANY = 96;                                   // candidates from which the best of them are chosen, so that the threshold rises
constexpr int BUFFER = MANY + PUSHERS * PER_THREAD;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
    const void *logits;
    long long ld; // entries between rows
    int rows, vocab, top;
    const int *targets;
    float *logprobs, *entropy, *top_logprobs;
    int *top_ids;
};

__device__ __forceinline__ u64 key_of(float x, unsigned index) {
    const unsigned b = __float_as_uint(x + 0.0f); // (-0 and 0 are equal)
    return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | ~index;
}
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ unsigned index_of(u64 key) { return ~(unsigned)key; }

__device__ __forceinline__ float ex2(float x) { // 2^x
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (a - ref) LOG2E of two entries in two instructions
__device__ __forceinline__ float2 scaled(float a, float b, float ref) {
    float2 y;
    asm("{.reg .b64 x, r, l; mov.b64 x, {%2, %3}; mov.b64 r, {%4, %4}; mov.b64 l, {%5, %5}; add.rn.f32x2 x, x, r; mul.rn.f32x2 x, x, l; mov.b64 {%0, %1}, x;}"
        : "=f"(y.x), "=f"(y.y) : "f"(a), "f"(b), "f"(-ref), "f"(LOG2E));
    return y;
}

struct Sum { // of a set of entries: its largest, and what the others add (s in units of log2)
    float m, z, s;
};
__device__ __forceinline__ Sum join(const Sum &p, const Sum &q) {
    const bool first = p.m >= q.m;
    const Sum &a = first ? p : q, &b = first ? q : p;
    const float d = (b.m - a.m) * LOG2E; // (-inf where a set is empty; NaN where both are)
    Sum r = a;
    const float e = d > -CUDART_INF_F ? ex2(d) : 0.0f;
    if (e > 0.0f) { // (else b adds nothing, and d (1 + b.z) may pass FP32's range)
        r.z = fmaf(1.0f + b.z, e, a.z);
        r.s = fmaf(fmaf(d, 1.0f + b.z, b.s), e, a.s);
    }
    r.z += b.z - b.z; // a NaN stays one, wherever it was
    return r;
}

template <typename T> struct Load;
template <> struct Load<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ void vec(const float *p, float *x) {
        const float4 v = __ldcs(reinterpret_cast<const float4 *>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
};
template <> struct Load<__half> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void vec(const __half *p, float *x) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(p));
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
};
template <> struct Load<bf16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void vec(const bf16 *p, float *x) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(p));
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ float one(const bf16 *p) { return __bfloat162float(*p); }
};

struct Smem {
    u64 buffer[BUFFER], best[MAX_TOP]; // candidates; the CTA's alternatives in order
    Sum warps[THREADS / 32], cta, parts[MAX_CLUSTER];
    int counts[MAX_CLUSTER];
    u64 merged[MAX_TOP];
    int pushed, n_best;
};

// The `n` largest keys of buffer[0 .. total), in order, into best: a key's place is the number of larger ones.
__device__ __forceinline__ void select(Smem &sm, int total, int n) {
    for (int i = threadIdx.x; i < total; i += THREADS) {
        const u64 k = sm.buffer[i];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < total; j++) place += sm.buffer[j] > k;
        if (place < n) sm.best[place] = k;
    }
    __syncthreads();
    const int kept = min(total, n);
    if (threadIdx.x < kept) sm.buffer[threadIdx.x] = sm.best[threadIdx.x];
    if (threadIdx.x == 0) sm.pushed = sm.n_best = kept;
    __syncthreads();
}

// A cluster of CTAs reads a row, each a stretch of it in batches of 16 entries a thread, the next batch under way while one is worked on.  A warp keeps the largest entry it has met and
// a thread the sum of its own entries in units of that; candidates for the alternatives are the entries above a threshold that at least `top` known ones reach, so that after the first
// batch hardly any is looked at twice.  Bytes are its floor: 512 rows of 128256 FP32 logits are 263 MB, 41 us; with
// 20 alternatives it takes 75 (3.5 TB/s), of which a CTA's selections are the part above a plain pass.  One such row with 5: 16 us, a cluster of 8, latency.
template <typename T> __global__ void __launch_bounds__(THREADS, 4) k_log_probs(const Args a) {
    constexpr int VEC = Load<T>::VEC;
    __shared__ Smem sm;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31;
    const T *x = (const T *)a.logits + row * a.ld;
    const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)); // entries between the 16-byte boundary in front of the row and its start
    const int span = skew + a.vocab; // (vocabularies of up to 2^30)
    // stretches of whole vectors, as even as that allows
    const int vecs = (span + VEC - 1) / VEC, begin = (int)((long long)vecs * rank / ranks) * VEC, end = (int)((long long)vecs * (rank + 1) / ranks) * VEC;
    if (tid == 0) { sm.pushed = 0; sm.n_best = 0; }
    float m = -CUDART_INF_F, z = 0.0f, s = 0.0f; // the warp's largest; this thread's sums, without it
    bool open = true;                // no bar yet: every entry is a candidate
    float bar_value = -CUDART_INF_F; // entries that are not larger are none
    const auto room = [&](float &value) { // in front of a batch's candidates, the same for every thread (a barrier follows the last ones): room for them, and a higher bar
        if (sm.pushed <= MANY) return;
        __syncthreads();
        select(sm, sm.pushed, a.top);
        if (sm.n_best == a.top) {
            open = false;
            value = fmaxf(value, value_of(sm.buffer[a.top - 1]));
        }
    };
    const auto fetch = [&](int base, float (&v)[PER_THREAD]) {
        const int from = base + tid * VEC - skew; // index in the row
        if (base >= skew && base + BATCH <= end && base + BATCH <= span) {
#pragma unroll
            for (int i = 0; i < PER_THREAD / VEC; i++) Load<T>::vec(x + from + i * (THREADS * VEC), v + i * VEC);
        } else
#pragma unroll
            for (int i = 0; i < PER_THREAD; i++) {
                const int at = from + i / VEC * (THREADS * VEC) + i % VEC;
                v[i] = at >= 0 && at < a.vocab && at + skew < end ? Load<T>::one(x + at) : -CUDART_INF_F;
            }
    };
    const auto take = [&](int base, const float (&v)[PER_THREAD]) {
        float top = v[0];
#pragma unroll
        for (int i = 1; i < PER_THREAD; i++) top = fmaxf(top, v[i]);
        const float widest = value_of((u64)__reduce_max_sync(0xffffffffu, (unsigned)(key_of(top == top ? top : -CUDART_INF_F, 0) >> 32)) << 32); // (all NaN: none)
        int skip = PER_THREAD; // this thread's entry that is the warp's largest from now on
        if (widest > m) {
            const float d = (m - widest) * LOG2E, e = d > -CUDART_INF_F ? ex2(d) : 0.0f;
            if (e > 0.0f) s = fmaf(d, z, s) * e; else s = 0.0f;
            z = z == z ? z * e : z;
            if (lane == 0 && e > 0.0f) { // the largest so far becomes one of the others
                z += e;
                s = fmaf(d, e, s);
            }
            m = widest;
            const unsigned owner = __ballot_sync(0xffffffffu, top == widest);
            if (lane == __ffs(owner) - 1)
#pragma unroll
                for (int i = PER_THREAD - 1; i >= 0; i--)
                    if (v[i] == widest) skip = i;
        }
        // x - m first: it is exact near m, so that neither a row's offset (with m LOG2E rounded, 2^-24 of that) nor a mask of the type's lowest value, whose m LOG2E overflows, is in y
        const float ref = m == -CUDART_INF_F ? 0.0f : m;
        float zs[2] = {0.0f, 0.0f}, ss[2] = {0.0f, 0.0f};
        if (__any_sync(0xffffffffu, skip < PER_THREAD)) {
#pragma unroll
            for (int i = 0; i < PER_THREAD; i += 2) {
                const float2 y = scaled(v[i], v[i + 1], ref);
                const float e0 = i == skip ? 0.0f : ex2(y.x), e1 = i + 1 == skip ? 0.0f : ex2(y.y);
                zs[0] += e0;
                zs[1] += e1;
                ss[0] = fmaf(fmaxf(y.x, -1000.0f), e0, ss[0]); // (-inf times 0 is none)
                ss[1] = fmaf(fmaxf(y.y, -1000.0f), e1, ss[1]);
            }
        } else
#pragma unroll
            for (int i = 0; i < PER_THREAD; i += 2) {
                const float2 y = scaled(v[i], v[i + 1], ref);
                const float e0 = ex2(y.x), e1 = ex2(y.y);
                zs[0] += e0;
                zs[1] += e1;
                ss[0] = fmaf(fmaxf(y.x, -1000.0f), e0, ss[0]);
                ss[1] = fmaf(fmaxf(y.y, -1000.0f), e1, ss[1]);
            }
        z += zs[0] + zs[1];
        s += ss[0] + ss[1];
        if (a.top == 0) return;
        const auto index = [&](int i) { return base + i / VEC * (THREADS * VEC) + tid * VEC + i % VEC - skew; };
        if (!open) { // `top` entries of earlier batches reach the bar: equal ones, whose index is larger, do not beat them
            const bool over = top > bar_value;
            const int n = __syncthreads_count(over);
            if (n == 0) return;
            if (n <= PUSHERS) {
                room(bar_value);
                __syncthreads();
                if (over)
#pragma unroll
                    for (int i = 0; i < PER_THREAD; i++)
                        if (v[i] > bar_value) sm.buffer[atomicAdd(&sm.pushed, 1)] = key_of(v[i], (unsigned)index(i));
                return;
            }
        }
        // the first batch, and one that brings many: a bar that at least `top` and at most PUSHERS threads reach
        u64 largest = 0;
#pragma unroll
        for (int i = 0; i < PER_THREAD; i++) {
            const int at = index(i);
            if (at >= 0 && at < a.vocab && at + skew < end && v[i] == v[i]) {
                const u64 k = key_of(v[i], (unsigned)at);
                if (k > largest) largest = k;
            }
        }
        const bool over = open ? largest > 0 : top > bar_value;
        const int n = __syncthreads_count(over);
        u64 least = 1;
        float next = bar_value;
        if (n > PUSHERS) { // half the interval at a time; the keys are no two alike, so such a bar exists
            u64 low = 0, high = ~0ull;
            for (;;) {
                least = low + (high - low) / 2;
                const int above = __syncthreads_count(over && largest >= least);
                if (above > PUSHERS) low = least;
                else if (above < a.top) high = least;
                else break;
            }
            next = value_of(least);
            open = false;
        }
        room(next);
        __syncthreads();
        if (over && largest >= least)
#pragma unroll
            for (int i = 0; i < PER_THREAD; i++) {
                const int at = index(i);
                const u64 k = key_of(v[i], (unsigned)at);
                if (at >= 0 && at < a.vocab && at + skew < end && v[i] == v[i] && k >= least) sm.buffer[atomicAdd(&sm.pushed, 1)] = k;
            }
        bar_value = fmaxf(bar_value, next);
    };
    float now[PER_THREAD], next[PER_THREAD];
    if (begin < end) fetch(begin, next);
    __syncthreads();
#pragma unroll 1
    for (int base = begin; base < end; base += BATCH) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; i++) now[i] = next[i];
        if (base + BATCH < end) fetch(base + BATCH, next);
        take(base, now);
    }
    // ---- join: threads, then CTAs -------------------------------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) sm.warps[tid >> 5] = {m, z, s};
    __syncthreads();
    if (a.top) select(sm, sm.pushed, a.top);
    if (tid == 0) {
        Sum all = sm.warps[0];
        for (int w = 1; w < THREADS / 32; w++) all = join(all, sm.warps[w]);
        sm.cta = all;
    }
    if (ranks > 1) cluster.sync(); else __syncthreads();
    if (rank == 0) {
        if (tid < ranks) { // (a CTA a thread: one after the other, each is a trip to another SM)
            sm.parts[tid] = *cluster.map_shared_rank(&sm.cta, tid);
            sm.counts[tid] = *cluster.map_shared_rank(&sm.n_best, tid);
        }
        u64 mine = 0;
        static_assert(THREADS >= MAX_CLUSTER * MAX_TOP, "a key a thread");
        if (a.top && tid < ranks * MAX_TOP) mine = *cluster.map_shared_rank(&sm.best[tid % MAX_TOP], tid / MAX_TOP);
        __syncthreads();
        Sum all = sm.parts[0];
        for (int r = 1; r < ranks; r++) all = join(all, sm.parts[r]);
        const float log_z = all.m < CUDART_INF_F ? log1pf(all.z) : CUDART_NAN_F; // (an infinite logit, or none that is not -inf)
        const float inv = 1.0f / (1.0f + all.z);
        const bool none = !(all.m > -CUDART_INF_F);
        if (tid == 0) {
            if (a.logprobs) {
                const int t = a.targets ? a.targets[row] : -1;
                a.logprobs[row] = t < 0 || t >= a.vocab ? 0.0f : none ? CUDART_NAN_F : Load<T>::one(x + t) - all.m - log_z;
            }
            if (a.entropy) a.entropy[row] = none ? CUDART_NAN_F : log_z - all.s * LN2 * inv;
        }
        if (a.top) {
            u64 *all_keys = sm.buffer; // every CTA's alternatives, in order: [rank][MAX_TOP]; 0 behind the last
            static_assert(BUFFER >= MAX_CLUSTER * MAX_TOP, "the lists of all CTAs");
            if (tid < ranks * MAX_TOP) all_keys[tid] = mine = tid % MAX_TOP < sm.counts[tid / MAX_TOP] ? mine : 0;
            __syncthreads();
            if (mine) {
                int place = 0;
                for (int q = 0; q < ranks; q++) { // half of a list at a time
                    const u64 *best = all_keys + q * MAX_TOP;
                    int low = 0;
#pragma unroll
                    for (int step = MAX_TOP / 2; step > 0; step /= 2)
                        if (best[low + step - 1] > mine) low += step;
                    place += low + (best[low] > mine);
                }
                if (place < a.top) sm.merged[place] = mine;
            }
            int have = 0;
            for (int r = 0; r < ranks; r++) have += sm.counts[r];
            __syncthreads();
            if (tid < a.top) { // fewer than `top` numbers in the row: -1
                const bool is = tid < have;
                const u64 k = is ? sm.merged[tid] : 0;
                if (a.top_ids) a.top_ids[(size_t)row * a.top + tid] = is ? (int)index_of(k) : -1;
                if (a.top_logprobs) a.top_logprobs[(size_t)row * a.top + tid] = none || !is ? CUDART_NAN_F : value_of(k) - all.m - log_z;
            }
        }
    }
    if (ranks > 1) cluster.sync(); // no CTA leaves while the first one reads its part
}

} // namespace lp
