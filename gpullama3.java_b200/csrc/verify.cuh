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
// Nothing depends on an order of arrival.
#pragma once
#include "logprobs.cuh"

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

// A stretch is read whole into registers: largest entry, then the sum.  FP32: an exponential's argument is off by at most 2^-24 of itself, so a row's sum by sum p |log2 p| 2^-24 and 2^-20 for
// the exponentials and the order of the sum: 3e-6 at most.
template <typename T> __global__ void __launch_bounds__(ROW_THREADS, 5) k_verify_rows(const Args a) {
    constexpr int VEC = Load<T>::VEC;
    __shared__ float warp_top[ROW_THREADS / 32], warp_sum[ROW_THREADS / 32];
    __shared__ int warp_at[ROW_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
// 64-bit sums of weights over the vocabulary, by warp, CTA and cluster.
struct Sums {
    double warp[TOKEN_WARPS], cta[CLUSTER]; // this CTA's warps; every CTA
};

template <typename T> __global__ void __launch_bounds__(TOKEN_THREADS) k_verify_token(const Args a) {
    constexpr int VEC = Load<T>::VEC;
    __shared__ Row rows[2 * MAX_DRAFTS + 1]; // target rows, then draft rows
    __shared__ signed char verdict[MAX_DRAFTS]; // 1 accepted, 0 not, -1 too close, -2 no distribution
    __shared__ Sums sums[2];
    __shared__ double scan[TOKEN_WARPS];
    __shared__ int found;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank(), s = blockIdx.x / CLUSTER;
    pdl_wait();
    cluster.sync(); // every CTA is there before another writes into its memory
    const int c = given(a, s, a.drafts);
    const int *d = a.tokens + (long long)s * a.drafts;
    const float *u = a.uniforms + (long long)s * (a.drafts + 1);
    const int greedy = a.greedy, both = a.both;
    const float to_log2 = greedy ? 0.0f : LOG2E / a.temperature;
    const double inv_t = greedy ? 0.0 : 1.0 / (double)a.temperature;
    const auto target = [&](int i) { return (const T *)a.logits + s * a.ld_s + i * a.ld_r; };
    const auto draft = [&](int i) { return (const T *)a.draft_logits + s * a.draft_ld_s + i * a.draft_ld_r; };

    // ---- the rows' parts, a row a warp ----
    for (int r = warp; r < (both ? 2 * c + 1 : c + 1); r += TOKEN_WARPS) {
        const bool first = r <= c;
        const size_t row = first ? (size_t)s * (a.drafts + 1) + r : (size_t)a.sequences * (a.drafts + 1) + (size_t)s * a.drafts + r - c - 1;
        float top = -CUDART_INF_F;
        for (int j = lane; j < a.stretches; j += 32) top = fmaxf(top, a.parts[row * a.stretches + j].top);
        top = warp_max_f(top);
        double sum = 0.0;
        int at = INT_MAX;
        bool nan = false;
        for (int j = lane; j < a.stretches; j += 32) {
            const Part p = a.parts[row * a.stretches + j];
            nan |= p.sum != p.sum;
            if (p.top == -CUDART_INF_F) continue;
            sum += (double)p.sum * (double)(p.top == top ? 1.0f : ex2((p.top - top) * to_log2));
            if (p.top == top) at = min(at, p.at);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        at = __reduce_min_sync(0xffffffffu, at);
        nan = __any_sync(0xffffffffu, nan);
        if (lane == 0) rows[first ? r : MAX_DRAFTS + r - c] = {top, at, nan || !(fabsf(top) < CUDART_INF_F) ? -1.0 : greedy ? 1.0 : sum};
    }
    __syncthreads();
    const auto of_draft = [&](int i) -> Row & { return rows[MAX_DRAFTS + 1 + i]; };
    const auto chance = [&](const Row &r, const T *x, int j) { return exp(((double)Load<T>::one(x + j) - (double)r.top) * inv_t) / r.sum; };
    const auto decide = [&](int i) { // u q < p, and by how much
        const Row &p = rows[i];
        if (!(p.sum > 0.0) || (both && !(of_draft(i).sum > 0.0))) return -2;
        if (greedy) return p.at == d[i] ? 1 : 0;
        const double x = (double)u[i] * (both ? chance(of_draft(i), draft(i), d[i]) : 1.0), y = chance(p, target(i), d[i]);
        return fabs(x - y) <= 1e-5 * fmax(x, y) && y > 0.0 ? -1 : x < y ? 1 : 0;
    };
    if (tid < c) verdict[tid] = (signed char)decide(tid);
    __syncthreads();

    // Sums of weights f(j, x_j, y_j) over the vocabulary, which the cluster's warps share in order; y may be null.
    const int share = ((a.vocab + CLUSTER * TOKEN_WARPS - 1) / (CLUSTER * TOKEN_WARPS) + 7) / 8 * 8; // (whole vectors)
    const auto begin_of = [&](int w) { return (int)min((long long)w * share, (long long)a.vocab); };
    const auto add = [&](Sums &to, const T *x, const T *y, auto f) {
        const int begin = begin_of(rank * TOKEN_WARPS + warp), end = begin_of(rank * TOKEN_WARPS + warp + 1);
        double sum = 0.0;
        for (int j0 = begin; j0 < end; j0 += 2 * 32 * VEC) {
            float p[2][VEC], q[2][VEC];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int j = j0 + (h * 32 + lane) * VEC;
                if (a.vec && j + VEC <= end) {
                    Load<T>::vec(x + j, p[h]);
                    if (y) Load<T>::vec(y + j, q[h]);
                } else
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        p[h][k] = j + k < end ? Load<T>::one(x + j + k) : -CUDART_INF_F;
                        q[h][k] = y && j + k < end ? Load<T>::one(y + j + k) : -CUDART_INF_F;
                    }
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int k = 0; k < VEC; k++) sum += f(j0 + (h * 32 + lane) * VEC + k, p[h][k], y ? q[h][k] : 0.0f);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) to.warp[warp] = sum;
        __syncthreads();
        if (tid < CLUSTER) { // to every CTA of the cluster
            double cta = 0.0;
#pragma unroll
            for (int w = 0; w < TOKEN_WARPS; w++) cta += to.warp[w];
            *cluster.map_shared_rank(&to.cta[rank], tid) = cta;
        }
        cluster.sync();
        double all = 0.0;
#pragma unroll
        for (int r = 0; r < CLUSTER; r++) all += to.cta[r];
        return all;
    };
    const auto weight = [&](const Row &r, float x) { return exp(((double)x - (double)r.top) * inv_t); };

    int n = 0;
    bool fails = false;
    for (; n < c; n++) {
        int v = verdict[n];
        if (v == -1) { // (all CTAs of the cluster come to the same)
            Row &p = rows[n];
            const Row was = p;
            const double sp = add(sums[0], target(n), (const T *)nullptr, [&](int, float x, float) { return weight(was, x); });
            double sq = 1.0;
            if (both) {
                const Row wasq = of_draft(n);
                sq = add(sums[1], draft(n), (const T *)nullptr, [&](int, float x, float) { return weight(wasq, x); });
            }
            const double x = (double)u[n] * (both ? exp(((double)Load<T>::one(draft(n) + d[n]) - (double)of_draft(n).top) * inv_t) / sq : 1.0);
            v = x < exp(((double)Load<T>::one(target(n) + d[n]) - (double)was.top) * inv_t) / sp;
            cluster.sync(); // (the sums' memory is used again)
        }
        fails = v == -2;
        if (v != 1) break;
    }
    if (n == c) fails = !(rows[c].sum > 0.0);
    if (rank == 0) {
        for (int i = tid; i <= a.drafts; i += TOKEN_THREADS)
            if (i != n) a.out_tokens[(long long)s * (a.drafts + 1) + i] = i < n ? d[i] : -1;
        if (tid == 0) {
            a.accepted[s] = n;
            if (fails || greedy) a.out_tokens[(long long)s * (a.drafts + 1) + n] = fails ? -1 : rows[n].at;
        }
    }
    if (fails || greedy) return; // (the same in every CTA of the cluster)

    // ---- the token ----
    const bool left = n < c; // a draft that did not stand
    const Row p = rows[n], q = rows[both && left ? MAX_DRAFTS + 1 + n : n];
    const int without = left && !both ? d[n] : -1; // it was looked up
    const auto whole = [&](int, float x, float) { return weight(p, x); };
    const auto rest = [&](int j, float x, float) { return j == without ? 0.0 : weight(p, x); };
    double total = add(sums[0], target(n), (const T *)nullptr, rest), sp = total, sq = 1.0;
    int kind = 0; // of weights: rest, difference, whole
    Sums *by = &sums[0];
    if (both && left) {
        sq = add(sums[1], draft(n), (const T *)nullptr, [&](int, float x, float) { return weight(q, x); });
        cluster.sync();
        const auto more = [&](int, float x, float y) { return fmax(weight(p, x) / sp - weight(q, y) / sq, 0.0); };
        total = add(sums[1], target(n), draft(n), more);
        by = &sums[1];
        kind = 1;
        if (!(total > 0.0)) { // the same distributions
            by = &sums[0];
            kind = 0;
            total = sp;
        }
    } else if (without >= 0 && !(total > 0.0)) { // nothing but the draft
        cluster.sync();
        total = add(sums[0], target(n), (const T *)nullptr, whole);
        kind = 2;
    }
    const auto one = [&](int j) -> double {
        const float x = Load<T>::one(target(n) + j);
        return kind == 1 ? fmax(weight(p, x) / sp - weight(q, Load<T>::one(draft(n) + j)) / sq, 0.0) : kind == 0 ? rest(j, x, 0.0f) : whole(j, x, 0.0f);
    };
    // which CTA, which warp's share, which entry: the first whose running sum passes the border, or the last that weighs anything
    const double border = (double)u[a.drafts] * total;
    double before = 0.0, sum = 0.0;
    int chosen = -1;
    for (int r = 0; r < CLUSTER; r++) {
        const double x = by->cta[r];
        if (x > 0.0) { chosen = r; before = sum; }
        sum += x;
        if (x > 0.0 && sum > border) break;
    }
    if (chosen == rank) { // (the others are done: nothing of theirs is read any more)
        int w_chosen = 0;
        double at = before;
        sum = before;
        for (int w = 0; w < TOKEN_WARPS; w++) {
            const double x = by->warp[w];
            if (x > 0.0) { w_chosen = w; at = sum; }
            sum += x;
            if (x > 0.0 && sum > border) break;
        }
        const int begin = begin_of(rank * TOKEN_WARPS + w_chosen), end = begin_of(rank * TOKEN_WARPS + w_chosen + 1);
        int last = -1; // this thread's last entry that weighs anything
        if (tid == 0) found = INT_MAX;
        __syncthreads();
        for (int j0 = begin; j0 < end; j0 += TOKEN_THREADS) {
            const int j = j0 + tid;
            const double x = j < end ? one(j) : 0.0;
            double run = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += y;
            }
            if (lane == 31) scan[warp] = run;
            __syncthreads();
            double front = at, all = at;
#pragma unroll
            for (int w = 0; w < TOKEN_WARPS; w++) {
                if (w == warp) front = all;
                all += scan[w];
            }
            if (x > 0.0) last = j;
            if (x > 0.0 && front + run > border) atomicMin(&found, j);
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
        }
        if (tid == 0) a.out_tokens[(long long)s * (a.drafts + 1) + n] = found;
    }
}

} // namespace verify
