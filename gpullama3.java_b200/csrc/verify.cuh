// verify.cuh -- how many drafted tokens stand against the target's distributions, and the token behind them, from given uniform numbers.
//
// Of a sequence: target rows x_0 .. x_K, drafts d_1 .. d_c (c <= K: the first that is no token ends them), p_i = softmax(x_i / T), q_i = softmax(y_i / T) of the draft's logits, or all on
// d_i where a draft was looked up.  Draft i + 1 is accepted when u_{i+1} q_i(d) < p_i(d); n is the first that is not, or c.  The token comes from weights w: p_c where all were accepted, else
// max(p_n - q_n, 0) (p_n without d); all of them 0: p_n.  It is the first index whose running sum passes u sum(w).  T = 0: a draft is accepted when it is the row's largest (the first
// of equal ones), and that is the token.
//
// k_verify_rows reads every row once: a CTA a stretch of it, its largest entry and the sum of exp((x - largest) / T) in FP32.  k_verify_token, a cluster a sequence, joins them, decides, and
// draws the token: that is a whole number which one more bit would change where u falls near a border, and a vocabulary has 10^5 of them, so the drawn row's weights and their sums are in
// 64 bits; and where FP32's error could turn a decision, its row's sum is taken once more in 64 bits.
// Where the token comes from max(p - q, 0), one pass takes both rows' sums and, on either side of which p / sum_p > q / sum_q by FP32's sums, those of the entries that weigh more in p: their difference is the
// weight (entries that weigh the same to 2^-40 weigh nothing; a pass for the sums and one for the weights took 70 us in place of 37).  An entry whose weights agree to FP32's error, 8e-6, may be counted on the wrong
// side, by a difference of no more than that of itself: a border moves by 8e-6 of such entries' p.
// Bytes are the floor: 32 sequences of 0 to 5 drafts, 84 in all, and 128256 FP32 logits of two models: 200 rows that count, 103 MB, 15.9 us; the call takes 53-55 (48 in a graph): the rows 23, the tokens 24-34, of
// which a pass over two rows in 64 bits is 18: two exponentials an entry, 64-bit units at 23 % on average, their chains and the loads in between on the clusters that have one.  One sequence: 15.7 in a graph, latency.
// Nothing depends on an order of arrival.
#pragma once
#include "kv4.cuh"
#include "logprobs.cuh"

#include <string.h>

namespace verify {

namespace cg = cooperative_groups;
using lp::bf16;
using lp::ex2;
using lp::Load;
using lp::LOG2E;

constexpr int ROW_THREADS = 256, ROW_ENTRIES = 32, STRETCH = ROW_THREADS * ROW_ENTRIES; // entries of a CTA
constexpr int TOKEN_THREADS = 512, TOKEN_WARPS = TOKEN_THREADS / 32, CLUSTER = 8, MAX_DRAFTS = 64;

struct Part { // of a stretch: its largest entry and that one's index, the sum (NaN where an entry is)
    float top, sum;
    int at, unused;
};
struct Args {
    const void *logits, *draft_logits; // rows (sequence, i): sequence * ld_s + i * ld_r
    long long ld_s, ld_r, draft_ld_s, draft_ld_r;
    int sequences, drafts, vocab, stretches;
    int vec, greedy, both; // every row starts on a 16-byte boundary; temperature 0; there are draft logits, and they count
    float temperature;
    const int *tokens;
    const float *uniforms;
    int *out_tokens, *accepted;
    Part *parts; // [target rows, then draft rows][stretch]
};

__host__ __device__ inline int share_of(int vocab) { return ((vocab + CLUSTER * TOKEN_WARPS - 1) / (CLUSTER * TOKEN_WARPS) + 7) / 8 * 8; } // entries of a warp: whole vectors

// Drafts of a sequence in front of the first that is no token (at most `most` looked at): a warp.
__device__ __forceinline__ int given(const Args &a, int s, int most) {
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < most; i += 32) {
        const int d = i + lane < most ? a.tokens[(long long)s * a.drafts + i + lane] : -1;
        const unsigned ok = __ballot_sync(0xffffffffu, d >= 0 && d < a.vocab);
        if (ok != 0xffffffffu) return min(most, i + __ffs(~ok) - 1);
    }
    return most;
}

// A stretch is read whole into registers, so that all of its loads are under way at once: largest entry, then the sum.  FP32: an exponential's argument, distance times log2(e) / T, is off by at most 4 of 2^-24 of itself, so a row's sum by 4 ln(2) 2^-24 of
// their mean, which a vocabulary of 2^24 keeps below 20, and 2^-20 for the exponentials and the order of the sum: 4e-6 at most.
template <typename T> __global__ void __launch_bounds__(ROW_THREADS, 5) k_verify_rows(const Args a) {
    constexpr int VEC = Load<T>::VEC;
    __shared__ float warp_top[ROW_THREADS / 32], warp_sum[ROW_THREADS / 32];
    __shared__ int warp_at[ROW_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    const int row = blockIdx.x / a.stretches, stretch = blockIdx.x % a.stretches, per = a.drafts + 1, n_target = a.sequences * per;
    const bool target = row < n_target;
    const int s = target ? row / per : (row - n_target) / a.drafts, i = target ? row % per : (row - n_target) % a.drafts;
    const int needs = target ? i : i + 1; // drafts in front of it without which the row does not count
    if (needs && given(a, s, needs) < needs) return;
    const T *x = target ? (const T *)a.logits + s * a.ld_s + i * a.ld_r : (const T *)a.draft_logits + s * a.draft_ld_s + i * a.draft_ld_r;
    const int begin = stretch * STRETCH, count = min(STRETCH, a.vocab - begin);
    x += begin;
    float v[ROW_ENTRIES];
#pragma unroll
    for (int u = 0; u < ROW_ENTRIES; u += VEC) {
        const int j = (u / VEC * ROW_THREADS + tid) * VEC;
        if (a.vec && j + VEC <= count) Load<T>::vec(x + j, v + u);
        else
#pragma unroll
            for (int k = 0; k < VEC; k++) v[u + k] = j + k < count ? Load<T>::one(x + j + k) : -CUDART_INF_F;
    }
    float top = -CUDART_INF_F;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < ROW_ENTRIES; u++) {
        top = fmaxf(top, v[u]);
        nan |= v[u] != v[u];
    }
    const float mine = top;
    top = warp_max_f(top);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = warp_top[0];
#pragma unroll
    for (int w = 1; w < ROW_THREADS / 32; w++) top = fmaxf(top, warp_top[w]);
    float sum = 0.0f;
    int at = INT_MAX;
    if (a.greedy) {
        if (mine == top)
#pragma unroll
            for (int u = ROW_ENTRIES - 1; u >= 0; u--)
                if (v[u] == top) at = (u / VEC * ROW_THREADS + tid) * VEC + u % VEC; // (a thread's entries rise with u)
        at = __reduce_min_sync(0xffffffffu, at);
    } else {
        const float c = LOG2E / a.temperature, base = top == -CUDART_INF_F ? 0.0f : top;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < ROW_ENTRIES; u++) part[u & 3] += ex2((v[u] - base) * c);
        sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (__any_sync(0xffffffffu, nan)) sum = CUDART_NAN_F;
    if (lane == 0) { warp_sum[warp] = sum; warp_at[warp] = at; }
    __syncthreads();
    if (tid == 0) {
        sum = 0.0f;
        at = INT_MAX;
#pragma unroll
        for (int w = 0; w < ROW_THREADS / 32; w++) { sum += warp_sum[w]; at = min(at, warp_at[w]); }
        a.parts[(size_t)row * a.stretches + stretch] = {top, sum, at == INT_MAX ? INT_MAX : begin + at, 0};
    }
}

struct Row { // a row's largest entry and its sum; without a distribution: a sum that is not above 0
    float top;
    int at;
    double sum;
};
// The parts of a row joined: a warp.
__device__ __forceinline__ Row join_parts(const Args &a, size_t row, float to_log2) {
    const int lane = threadIdx.x & 31;
    float top = -CUDART_INF_F;
    double sum = 0.0;
    int at = INT_MAX;
    bool nan = false;
    for (int j = lane; j < a.stretches; j += 32) {
        const Part p = a.parts[row * a.stretches + j];
        nan |= p.sum != p.sum;
        if (p.top > top) {
            sum *= (double)ex2((top - p.top) * to_log2);
            top = p.top;
            at = p.at;
            sum += (double)p.sum;
        } else if (p.top > -CUDART_INF_F) sum += (double)p.sum * (double)(p.top == top ? 1.0f : ex2((p.top - top) * to_log2));
    }
    const float all = warp_max_f(top);
    sum = top == -CUDART_INF_F ? 0.0 : sum * (double)(top == all ? 1.0f : ex2((top - all) * to_log2));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    at = __reduce_min_sync(0xffffffffu, top == all ? at : INT_MAX);
    nan = __any_sync(0xffffffffu, nan);
    return {all, at, nan || !(fabsf(all) < CUDART_INF_F) ? -1.0 : a.greedy ? 1.0 : sum};
}

// Temperature 0: a CTA a sequence, a row a warp.
__global__ void __launch_bounds__(256) k_verify_greedy(const Args a) {
    __shared__ int best[MAX_DRAFTS + 1];
    pdl_wait();
    const int tid = threadIdx.x, s = blockIdx.x, c = given(a, s, a.drafts);
    const long long out = (long long)s * (a.drafts + 1);
    for (int r = tid / 32; r <= c; r += 8) {
        const Row row = join_parts(a, (size_t)out + r, 0.0f);
        if (tid % 32 == 0) best[r] = row.sum > 0.0 ? row.at : -1;
    }
    __syncthreads();
    if (tid >= 32) return;
    int n = 0;
    while (n < c && best[n] == a.tokens[(long long)s * a.drafts + n]) n++;
    for (int i = tid; i <= a.drafts; i += 32) a.out_tokens[out + i] = i <= n ? best[i] : -1;
    if (tid == 0) a.accepted[s] = n;
}

// 64-bit sums over the vocabulary: of p = exp((x - top) / T), of q likewise, and of both where p weighs more.
constexpr int SUMS = 4;
struct Sums {
    double warp[SUMS][TOKEN_WARPS], cta[SUMS][CLUSTER]; // this CTA's warps; every CTA
};
__device__ __forceinline__ float4 load4(const float *x) { return __ldcs(reinterpret_cast<const float4 *>(x)); }
template <typename T> __device__ __forceinline__ float4 load4(const T *x) {
    const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(x));
    const float2 a = kv4::to_f32x2(w.x, x), b = kv4::to_f32x2(w.y, x);
    return make_float4(a.x, a.y, b.x, b.y);
}
// exp((x - top) / T) for x <= top: 2^(k / 32) from a table, the rest, at most ln(2) / 64, by its series (P. T. P. Tang's table-driven exponential, 1989).  Off by 4.5e-16 |x - top| / T (the argument: the difference,
// log2(e), the division by T and the product each round by 2^-53 of it) and 3e-15 of itself (the series leaves ln(2)^6 / 64^6 / 720 = 2.2e-15 out; table, series and product round): 3.2e-13 at the far end.  Below e^-690 it is 0, and whether it is is told by the
// 64-bit argument: x and top may be as large against T as they like (top - 690 T in FP32 would round to the neighbour of top, and let arguments in whose exponents leave the double's field).
constexpr int EXP_TABLE = 32;
// Weights of p and q that agree to 2^-40 are the same, so that what rounding leaves is not drawn from: 9.1e-13 is more than two far weights and the rows' sums (one after the other in a lane at most 2^10 numbers of
// the largest vocabulary: 1.2e-13 each) can be off, 8.8e-13.
constexpr double LOG2E_64 = 1.44269504088896340736, EVEN = 1.0 + 0x1p-40;
constexpr uint32_t REACH = 0x40df1badu;                                    // high word of 690 * 32 log2(e) = 31854.7
__host__ __device__ __forceinline__ uint32_t high_word(double v) {
#ifdef __CUDA_ARCH__
    return (uint32_t)__double2hiint(v);
#else
    uint64_t b;
    memcpy(&b, &v, 8);
    return (uint32_t)(b >> 32);
#endif
}
__host__ __device__ __forceinline__ uint32_t low_word(double v) {
#ifdef __CUDA_ARCH__
    return (uint32_t)__double2loint(v);
#else
    uint64_t b;
    memcpy(&b, &v, 8);
    return (uint32_t)b;
#endif
}
__host__ __device__ __forceinline__ double of_words(uint32_t high, uint32_t low) {
#ifdef __CUDA_ARCH__
    return __hiloint2double((int)high, (int)low);
#else
    const uint64_t b = (uint64_t)high << 32 | low;
    double v;
    memcpy(&v, &b, 8);
    return v;
#endif
}
__host__ __device__ inline double exp_scale(float temperature) { return EXP_TABLE * LOG2E_64 / (double)temperature; }
// table(i): 2^(i / 32); also on the host, where tests look at it
template <typename F> __host__ __device__ __forceinline__ double exp_of(float x, float top, double scale, F table) {
    constexpr double MAGIC = 6755399441055744.0, A = 0.693147180559945309417232 / EXP_TABLE; // 1.5 * 2^52: its last bits are those of the whole number added
    const double u = ((double)x - (double)top) * scale, d = u + MAGIC, r = u - (d - MAGIC);
    const uint32_t k = low_word(d);
    const double p = fma(fma(fma(fma(fma(A * A * A * A * A / 120.0, r, A * A * A * A / 24.0), r, A * A * A / 6.0), r, A * A / 2.0), r, A), r, 1.0) * table((int)(k & (EXP_TABLE - 1)));
    const bool some = (high_word(u) & 0x7fffffffu) <= REACH; // (not -inf)
    return of_words(some ? high_word(p) + ((uint32_t)((int)k >> 5) << 20) : 0u, some ? low_word(p) : 0u);
}
struct Weight {
    uint32_t table; // in shared memory: low, then high words of 2^(i / 32): 32 banks each, no conflicts
    double scale;   // 32 log2(e) / T
    __device__ __forceinline__ double operator()(float x, float top) const {
        return exp_of(x, top, scale, [&](int i) {
            uint32_t lo, hi;
            const uint32_t at = table + i * 4;
            asm("ld.shared.b32 %0, [%1];" : "=r"(lo) : "r"(at));
            asm("ld.shared.b32 %0, [%1 + 128];" : "=r"(hi) : "r"(at));
            return of_words(hi, lo);
        });
    }
};

// Passes over the rows of a draft or of the token: for a verdict; of weights p; of p - q; of p - q once more, by exact sums; of p whole.  Behind one for a verdict comes the next such or the
// token's first; behind the token's one with a higher number, or none any more.  So a sequence of c drafts takes c + 3 at most, whatever the sums are.
enum Pass { VERDICT = -1, TARGET = 0, MORE = 1, MORE_EXACT = 2, WHOLE = 3, DRAW = 4, NOTHING = 5 }; // DRAW: the token is drawn from this pass; NOTHING: there is nothing to draw from
__host__ __device__ __forceinline__ int after_pass(int kind, const double *all, double &sum_p, double &sum_q) { // all: the pass's sums; sum_p, sum_q: of the rows, exact ones behind MORE
    const bool some = all[0] > 0.0 && all[0] < 1e300;
    if (kind == TARGET) return some ? DRAW : WHOLE; // nothing but the draft: p as it is
    if (kind == WHOLE) return some ? DRAW : NOTHING;
    sum_p = all[0];
    sum_q = all[1];
    const double left = all[2] / sum_p - all[3] / sum_q;
    // Which entries weigh more was told by FP32's sums, each off by 4e-6 at most: an entry on the wrong side adds no more than twice that of itself, and few are that near.  Where little is left over they
    // might count.
    if (kind == MORE && !(left > 0.05)) return MORE_EXACT;
    return some && left > 0.0 && left < 2.0 ? DRAW : WHOLE; // (WHOLE: the same distributions)
}

template <typename T> __global__ void __launch_bounds__(TOKEN_THREADS, 2) k_verify_token(const Args a) {
    __shared__ Row rows[2 * MAX_DRAFTS + 1];    // target rows, then draft rows
    __shared__ signed char verdict[MAX_DRAFTS]; // 1 accepted, 0 not, -1 too close, -2 no distribution
    __shared__ Sums sums;
    __shared__ double scan[TOKEN_WARPS];
    __shared__ unsigned table[2][EXP_TABLE];
    __shared__ int found;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank(), s = blockIdx.x / CLUSTER;
    if (tid < EXP_TABLE) {
        const double x = exp2((double)tid / EXP_TABLE);
        table[0][tid] = (unsigned)__double2loint(x);
        table[1][tid] = (unsigned)__double2hiint(x);
    }
    const int c = given(a, s, a.drafts);
    const int *d = a.tokens + (long long)s * a.drafts;
    const float *u = a.uniforms + (long long)s * (a.drafts + 1);
    const int both = a.both;
    const Weight weight = {(uint32_t)__cvta_generic_to_shared(table), exp_scale(a.temperature)};
    const auto target = [&](int i) { return (const T *)a.logits + s * a.ld_s + i * a.ld_r; };
    const auto draft = [&](int i) { return (const T *)a.draft_logits + s * a.draft_ld_s + i * a.draft_ld_r; };
    cluster.sync(); // every CTA is there before another writes into its memory
    pdl_wait();

    // ---- the rows' parts, a row a warp ----
    for (int r = warp; r < (both ? 2 * c + 1 : c + 1); r += TOKEN_WARPS) {
        const bool first = r <= c;
        const Row row = join_parts(a, first ? (size_t)s * (a.drafts + 1) + r : (size_t)a.sequences * (a.drafts + 1) + (size_t)s * a.drafts + r - c - 1, LOG2E / a.temperature);
        if (lane == 0) rows[first ? r : MAX_DRAFTS + r - c] = row;
    }
    __syncthreads();
    const auto of_draft = [&](int i) -> Row & { return rows[MAX_DRAFTS + 1 + i]; };
    const auto decide = [&](int i, double sum, double draft_sum) { // u q < p; 2 and 3: too close for sums of FP32
        const double q = both ? weight(Load<T>::one(draft(i) + d[i]), of_draft(i).top) / draft_sum : 1.0;
        const double x = (double)u[i] * q, y = weight(Load<T>::one(target(i) + d[i]), rows[i].top) / sum;
        return fabs(x - y) <= 1e-5 * fmax(x, y) && y > 0.0 ? x < y ? 3 : 2 : x < y ? 1 : 0;
    };
    if (tid < c) {
        const int v = !(rows[tid].sum > 0.0) || (both && !(of_draft(tid).sum > 0.0)) ? -2 : decide(tid, rows[tid].sum, of_draft(tid).sum);
        verdict[tid] = (signed char)(v >= 2 ? -1 : v);
    }
    __syncthreads();

    // One pass over target row i, without entry `without`, and draft row i (two), which the cluster's warps share in order: sums of p, of q, and of both where p / sum_p > q / sum_q.
    const int share = share_of(a.vocab);
    const auto begin_of = [&](int w) { return (int)min((long long)w * share, (long long)a.vocab); };
    int n = 0, kind = VERDICT, without = -1;
    double sum_p = 1.0, sum_q = 1.0; // of the rows that the pass is for
    bool fails = true; // (until a pass is there to draw from)
    for (int pass = 0; pass < c + 3; pass++) {
        if (kind == VERDICT) { // the next draft whose verdict takes a pass, or the token
            int v = 1;
            while (n < c && (v = verdict[n]) == 1) n++;
            if (n < c ? v == -2 : !(rows[c].sum > 0.0)) break;
            if (n == c || v == 0) {
                kind = n < c && both ? MORE : TARGET;
                without = n < c && !both ? d[n] : -1; // a looked-up draft that did not stand
            }
        }
        const bool two = both && n < c;
        const T *x = target(n), *y = two ? draft(n) : nullptr;
        const float top_p = rows[n].top, top_q = two ? of_draft(n).top : 0.0f;
        if (kind != MORE_EXACT) {
            sum_p = rows[n].sum;
            sum_q = two ? of_draft(n).sum : 1.0;
        }
        const double edge = sum_p / sum_q * EVEN; // p / sum_p > q / sum_q where p > q edge
        double part[SUMS] = {0.0, 0.0, 0.0, 0.0};
        const int begin = begin_of(rank * TOKEN_WARPS + warp), end = begin_of(rank * TOKEN_WARPS + warp + 1);
        const float nothing = -CUDART_INF_F;
#pragma unroll 1
        for (int j0 = begin; j0 < end; j0 += 128) {
            const int j = j0 + lane * 4;
            float4 xs = make_float4(nothing, nothing, nothing, nothing), ys = xs;
            if (two) { // (needed last)
                if (a.vec && j + 4 <= end) ys = load4(y + j);
                else {
                    if (j < end) ys.x = Load<T>::one(y + j);
                    if (j + 1 < end) ys.y = Load<T>::one(y + j + 1);
                    if (j + 2 < end) ys.z = Load<T>::one(y + j + 2);
                    if (j + 3 < end) ys.w = Load<T>::one(y + j + 3);
                }
            }
            if (a.vec && j + 4 <= end) xs = load4(x + j);
            else {
                if (j < end) xs.x = Load<T>::one(x + j);
                if (j + 1 < end) xs.y = Load<T>::one(x + j + 1);
                if (j + 2 < end) xs.z = Load<T>::one(x + j + 2);
                if (j + 3 < end) xs.w = Load<T>::one(x + j + 3);
            }
            if (without >= j && without < j + 4) {
                if (without == j) xs.x = nothing;
                if (without == j + 1) xs.y = nothing;
                if (without == j + 2) xs.z = nothing;
                if (without == j + 3) xs.w = nothing;
            }
            const double p0 = weight(xs.x, top_p), p1 = weight(xs.y, top_p), p2 = weight(xs.z, top_p), p3 = weight(xs.w, top_p);
            part[0] += (p0 + p1) + (p2 + p3);
            if (two) {
                const auto also = [&](double p, float yi) {
                    const double q = weight(yi, top_q);
                    part[1] += q;
                    const bool more = p > q * edge;
                    part[2] += more ? p : 0.0;
                    part[3] += more ? q : 0.0;
                };
                also(p0, ys.x);
                also(p1, ys.y);
                also(p2, ys.z);
                also(p3, ys.w);
            }
        }
#pragma unroll
        for (int k = 0; k < SUMS; k++)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) part[k] += __shfl_xor_sync(0xffffffffu, part[k], o);
        cluster.sync(); // what was added before has been read
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < SUMS; k++) sums.warp[k][warp] = part[k];
        __syncthreads();
        if (tid < SUMS * CLUSTER) { // to every CTA of the cluster
            double cta = 0.0;
#pragma unroll
            for (int w = 0; w < TOKEN_WARPS; w++) cta += sums.warp[tid / CLUSTER][w];
            *cluster.map_shared_rank(&sums.cta[tid / CLUSTER][rank], tid % CLUSTER) = cta;
        }
        cluster.sync();
        double all[SUMS] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int r = 0; r < CLUSTER; r++)
#pragma unroll
            for (int k = 0; k < SUMS; k++) all[k] += sums.cta[k][r];
        // (all CTAs of the cluster come to the same)
        if (kind == VERDICT) {
            if (tid == 0) verdict[n] = (signed char)(decide(n, all[0], all[1]) & 1);
            __syncthreads();
        } else {
            const int next = after_pass(kind, all, sum_p, sum_q);
            fails = next != DRAW;
            if (next >= DRAW) break;
            kind = next;
            if (kind == WHOLE) without = -1;
        }
    }
    if (rank == 0) {
        for (int i = tid; i <= a.drafts; i += TOKEN_THREADS)
            if (i != n) a.out_tokens[(long long)s * (a.drafts + 1) + i] = i < n ? d[i] : -1;
        if (tid == 0) {
            a.accepted[s] = n;
            if (fails) a.out_tokens[(long long)s * (a.drafts + 1) + n] = -1;
        }
    }
    if (fails) return; // (the same in every CTA of the cluster)

    // ---- the token: which CTA, which warp's share, which entry: the first whose running sum passes the border, or the last that weighs anything ----
    const bool differ = kind == MORE || kind == MORE_EXACT;
    const double by_p = 1.0 / sum_p, by_q = 1.0 / sum_q;
    const auto weight_of = [&](const double *p, const double *more_p, const double *more_q, int i) { return differ ? more_p[i] * by_p - more_q[i] * by_q : p[i]; };
    const auto cta_weight = [&](int r) { return weight_of(sums.cta[0], sums.cta[2], sums.cta[3], r); };
    const auto warp_weight = [&](int w) { return weight_of(sums.warp[0], sums.warp[2], sums.warp[3], w); };
    const T *x = target(n), *y = differ ? draft(n) : nullptr;
    const float top_p = rows[n].top, top_q = differ ? of_draft(n).top : 0.0f;
    const auto one = [&](int j) -> double {
        const double p = j == without ? 0.0 : weight(Load<T>::one(x + j), top_p);
        if (!differ) return p;
        const double v = p * by_p, w = weight(Load<T>::one(y + j), top_q) * by_q;
        return v > w * EVEN ? v - w : 0.0;
    };
    double total = 0.0;
    for (int r = 0; r < CLUSTER; r++) total += cta_weight(r);
    const double border = (double)u[a.drafts] * total, least = differ ? total * 1e-13 : 0.0; // (what rounding leaves of a share where both weigh the same)
    double before = 0.0, sum = 0.0;
    int chosen = 0; // (some CTA writes the token in any case)
    for (int r = 0; r < CLUSTER; r++) {
        const double w = cta_weight(r);
        if (w > least) { chosen = r; before = sum; }
        sum += w;
        if (w > least && sum > border) break;
    }
    if (chosen != rank) return; // (the others are done: nothing of theirs is read any more)
    int w_chosen = 0;
    double at = before;
    sum = before;
    for (int w = 0; w < TOKEN_WARPS; w++) {
        const double v = warp_weight(w);
        if (v > least / TOKEN_WARPS) { w_chosen = w; at = sum; }
        sum += v;
        if (v > least / TOKEN_WARPS && sum > border) break;
    }
    const int begin = begin_of(rank * TOKEN_WARPS + w_chosen), end = begin_of(rank * TOKEN_WARPS + w_chosen + 1);
    int last = -1; // this thread's last entry that weighs anything
    if (tid == 0) found = INT_MAX;
    __syncthreads();
    for (int j0 = begin; j0 < end; j0 += TOKEN_THREADS) {
        const int j = j0 + tid;
        const double v = j < end ? one(j) : 0.0;
        double run = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double w = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += w;
        }
        if (lane == 31) scan[warp] = run;
        __syncthreads();
        double front = at, all = at;
#pragma unroll
        for (int w = 0; w < TOKEN_WARPS; w++) {
            if (w == warp) front = all;
            all += scan[w];
        }
        if (v > 0.0) last = j;
        if (v > 0.0 && front + run > border) atomicMin(&found, j);
        __syncthreads();
        at = all;
        if (found != INT_MAX) break;
    }
    if (found == INT_MAX) { // (the sums round apart by a last bit)
        __syncthreads();
        if (tid == 0) found = -1;
        __syncthreads();
        atomicMax(&found, last);
        __syncthreads();
        if (found < 0) { // (a share of nothing but rounding: the last entry of the row that weighs anything, or its largest)
            for (int j = tid; j < a.vocab; j += TOKEN_THREADS)
                if (one(j) > 0.0) last = j;
            __syncthreads();
            atomicMax(&found, last);
            __syncthreads();
            if (found < 0) {
                for (int j = tid; j < a.vocab; j += TOKEN_THREADS)
                    if (Load<T>::one(x + j) == top_p) last = j;
                __syncthreads();
                atomicMax(&found, last);
                __syncthreads();
            }
        }
    }
    if (tid == 0) a.out_tokens[(long long)s * (a.drafts + 1) + n] = found;
}

} // namespace verify
