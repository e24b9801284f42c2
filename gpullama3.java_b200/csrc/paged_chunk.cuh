// paged_chunk.cuh -- attention of prompt chunks over the pages on the 5th-generation tensor cores, with 16-bit results.
//
// A CTA takes 128 rows (tokens x query heads of one key/value head) and runs through the positions that any of them sees, 128 at a time:
//   warps 16-25  copy keys and values from their pages as they are, [position][entry] in swizzled rows: two warps for each of the three tiles of keys and two of values that there is room for
//   warp 26      issues S = Q K^T (both K-major) and O += P V (P from TMEM, V entry-major)
//   warps 0-15   exponentials, two threads a row; P in the cache's type takes the place of S; O is scaled where a row's maximum has grown by too much, which is rare
// Even and odd tiles are two streams with accumulators, maxima and sums of their own, each of eight warps, which the end joins: while one waits for its products the other computes.
// Rows of a tile may belong to several sequences and stand in any order: a run of tokens of one sequence is a segment, the tiles of all segments are one list, and a row masks what is not its own.
// Rounding: probabilities are one number of the cache's type (half a step: 2^-8 BF16, 2^-11 FP16), sums are FP32.  With FP16 they count from 2^7, so that those down to 2^-31 of a row's
// largest are kept.
// A row whose sums are not finite (a value that is infinite or NaN reaches every row of the tile as 0 * NaN, also those that do not see it; sums of large BF16 values) is computed once more at
// the end, by the whole CTA in FP32, from what it sees.
// Measured (512 tokens of 32 heads over 8 of 128, 8192 positions, 66.6 GFLOP, pages of 64): 90 us in a graph, 740 TFLOP/s, 45 % of the 1647 measured; floor 40.  128 CTAs leave 20 SMs idle.  Of a tile's 2300 cycles the
// products take 1490 to issue (1024 alone): their operands and the copies of the next tiles share the bandwidth of shared memory; exponentials keep their unit busy in 44 % of the cycles.  One group of warps for a
// tile's keys and values one after the other 100-102 us, a warp a place 104, two 100; what a row sees as bits in place of comparisons 92 (and 31 -> 22 us for three chunks of 111 tokens through a window of 500).
// Every wait is bounded: after half a second the CTA gives up, waits for its products under way, frees its tensor memory and writes NaN for its rows.
#pragma once
#include "kv4_chunk.cuh"
#include "paged.cuh"

namespace paged {

using namespace kv4; // barriers, products, tensor memory

constexpr int C_ROWS = 128, C_KEYS = 128, C_K = 3, C_V = 2, C_SOFTMAX = 16, C_PAIR = 2, C_COPY = (C_K + C_V) * C_PAIR, C_ISSUER = C_SOFTMAX + C_COPY, C_THREADS = (C_ISSUER + 1) * 32;
__host__ __device__ constexpr int c_tile_bytes(int hs) { return hs * C_KEYS * 2; }
__host__ __device__ constexpr int c_width(int hs) { return hs % 64 == 0 ? 64 : 32; } // entries of a swizzled row: 128 or 64 bytes
template <int HS> __device__ __forceinline__ uint32_t c_at(int r, int c) {          // of the 8 entries 8 c .. of row r in a tile
    constexpr int W = c_width(HS), P = W / 8;
    return (uint32_t)(c / P * (C_KEYS * W * 2) + r * (W * 2) + ((c % P ^ (W == 64 ? r & 7 : r >> 1 & 3)) << 4));
}
// K-major operands: rows of 128 (or 64) bytes, 8 rows apart 1024 (512).  Entry-major: 8 positions of 64 (32) entries are 1024 (512) bytes, the next 64 (32) entries a block of all positions on.
template <int HS> __device__ __forceinline__ uint64_t k_major(uint32_t a, int k) { // k: step of 16 entries
    constexpr int W = c_width(HS), P = W / 16;
    a += k / P * (C_KEYS * W * 2) + k % P * 32;
    return W == 64 ? desc128(a) : desc64(a);
}
template <int HS> __device__ __forceinline__ uint64_t entry_major(uint32_t a, int k) { // k: step of 16 positions
    constexpr uint64_t W = c_width(HS), LBO = C_KEYS * W * 2 >> 4, SBO = 8 * W * 2 >> 4;
    a += k * 16 * (uint32_t)W * 2;
    return (uint64_t)((a & 0x3ffffu) >> 4) | (LBO << 16) | (SBO << 32) | (1ull << 46) | ((W == 64 ? 2ull : 4ull) << 61);
}

struct CSegment { // a run of tokens of one sequence and the positions [begin, end) that any of them sees; tiles of all segments up to and with this one
    int sequence, begin, end, tiles;
};
struct CSmem { // behind the operands
    unsigned have[C_K][C_KEYS / 32]; // by stage of the keys: positions that have a page
    unsigned long long k_full[C_K], k_free[C_K], v_full[C_V], v_free[C_V];
    unsigned long long s_full[2], p_full[2], drained; // by stream
    unsigned long long pair[C_SOFTMAX / 2];           // the two warps that share a stream's rows
    unsigned tmem, bail, again[2], repeat[2];         // again: a row's maximum has to move; repeat: these are the scores of the tile before once more
    unsigned bad[C_ROWS / 32];                        // rows whose sums are not finite
    int n_segments;
    int seq[C_ROWS], pos[C_ROWS], segment[C_ROWS]; // by token
    float half_row[2][2][C_ROWS];                  // by stream: what the two threads of a row tell each other, their sums at the end
    float top[2][C_ROWS];
    float block[C_THREADS / 32];
    CSegment segments[C_ROWS];
};
__host__ __device__ constexpr size_t c_smem_bytes(int hs) { return 1024 + (1 + C_K + C_V) * c_tile_bytes(hs) + sizeof(CSmem); }
constexpr unsigned C_TRIES = 1u << 17;
template <bool SLEEP = true> __device__ __forceinline__ bool c_wait(const void *bar, unsigned parity, volatile unsigned *bail) { // false: given up
    const uint32_t b = kv4::s32(bar);
    for (unsigned i = 1; i < C_TRIES; i++) {
        if (bar_passed(b, parity)) return true;
        if (SLEEP) __nanosleep(20);
        if ((i & 1023u) == 0u && *bail) return false;
    }
    *bail = 1u;
    return false;
}
__device__ __forceinline__ float block_all(CSmem &sh, float v, bool sum) { // of all threads of the CTA; NaN is no maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = sum ? v + w : fmaxf(v, w);
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.block[threadIdx.x / 32] = v;
    __syncthreads();
    v = sh.block[0];
    for (int i = 1; i < C_THREADS / 32; i++) v = sum ? v + sh.block[i] : fmaxf(v, sh.block[i]);
    return v;
}

// GIVE_UP (tests): for their last wait, that for the products that end a stream, the warps of the rows wait for a barrier at which nobody arrives.
template <int HS, typename T, bool GIVE_UP = false> __global__ void __launch_bounds__(C_THREADS, 1) k_paged_chunk(const Step a) {
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr float LIFT = F16 ? 7.0f : 0.0f, TOO_MUCH = F16 ? 32768.0f : 256.0f; // a sum of a thread's 64 probabilities of a tile
    extern __shared__ unsigned char raw_smem[];
    unsigned char *smem = raw_smem + (-kv4::s32(raw_smem) & 1023u); // the operands' swizzle counts from 1024-byte boundaries
    unsigned char *sQ = smem, *sK = sQ + c_tile_bytes(HS), *sV = sK + C_K * c_tile_bytes(HS);
    CSmem &sh = *reinterpret_cast<CSmem *>(sV + C_V * c_tile_bytes(HS));
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int G = a.pool.kv_heads, mul = a.heads / G;
    const unsigned of = (65535u + mul) / mul; // r / mul = r of >> 16: exact, as r mul < 2^16
    const auto token_of = [&](int r) { return (int)(r * of >> 16); };
    const int units = (a.rows.n + a.tokens - 1) / a.tokens;
    const int split = blockIdx.x % a.splits, kvh = blockIdx.x / a.splits % G, unit = units - 1 - blockIdx.x / a.splits / G; // the last tokens, which see most, first
    const int token0 = unit * a.tokens, tokens = min(a.tokens, a.rows.n - token0);

    if (tid == 0) {
        for (int i = 0; i < C_K; i++) {
            bar_init(&sh.k_full[i], C_PAIR);
            bar_init(&sh.k_free[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            bar_init(&sh.v_full[i], C_PAIR);
            bar_init(&sh.v_free[i], 1);
            bar_init(&sh.s_full[i], 1);
            bar_init(&sh.p_full[i], C_SOFTMAX / 2);
            sh.again[i] = sh.repeat[i] = 0;
        }
        for (int i = 0; i < C_SOFTMAX / 2; i++) bar_init(&sh.pair[i], 2);
        bar_init(&sh.drained, 1);
        for (int i = 0; i < C_ROWS / 32; i++) sh.bad[i] = 0;
        sh.bail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C_SOFTMAX) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(kv4::s32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid < C_ROWS) {
        int seq = -1, pos = -1;
        if (tid < tokens) seq = a.rows.place(token0 + tid, pos);
        sh.seq[tid] = seq;
        sh.pos[tid] = max(pos, -1);
        sh.segment[tid] = -1;
    }
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u; // scores times a positive factor
    const float factor = a.scale == 0.0f ? 1.0f : fmaxf(fabsf(a.scale * 1.4426950408889634f), 1.17549435e-38f);
    for (int i = tid; i < C_ROWS * (HS / 8); i += C_THREADS) {
        const int r = i / (HS / 8), c = i % (HS / 8), token = token_of(r);
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (token < tokens && a.scale != 0.0f) {
            const uint16_t *q = (const uint16_t *)a.q + (long long)(token0 + token) * a.ldq + (size_t)(kvh * mul + r - token * mul) * HS + c * 8;
            if (a.vec) w = *reinterpret_cast<const uint4 *>(q);
            else w = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
        }
        sts128(kv4::s32(sQ) + c_at<HS>(r, c), w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
    }
    __syncthreads();
    if (warp == 0) { // one sequence for all, as inside a prompt: one segment
        bool same = sh.seq[0] >= 0;
        int from = INT_MAX, to = 0;
        for (int i = lane; i < tokens; i += 32) {
            int lo, hi;
            visible(sh.pos[i], a.window, lo, hi);
            same &= sh.seq[i] == sh.seq[0];
            if (hi > lo) { from = min(from, lo); to = max(to, hi); }
        }
        same = __all_sync(0xffffffffu, same);
        from = __reduce_min_sync(0xffffffffu, from);
        to = __reduce_max_sync(0xffffffffu, to);
        if (same) {
            if (to > 0)
                for (int i = lane; i < tokens; i += 32) sh.segment[i] = 0;
            if (lane == 0) {
                if (to > 0) sh.segments[0] = {sh.seq[0], from, to, (to - from + C_KEYS - 1) / C_KEYS};
                sh.n_segments = to > 0;
            }
        } else if (lane == 0) {
            int n = 0, total = 0;
            for (int i = 0; i < tokens;) {
                const int s = sh.seq[i];
                int j = i, from = INT_MAX, to = 0;
                for (; j < tokens && sh.seq[j] == s; j++) {
                    int lo, hi;
                    visible(sh.pos[j], a.window, lo, hi);
                    if (hi > lo) { from = min(from, lo); to = max(to, hi); }
                }
                if (s >= 0 && to > 0) {
                    total += (to - from + C_KEYS - 1) / C_KEYS;
                    for (int k = i; k < j; k++) sh.segment[k] = n;
                    sh.segments[n++] = {s, from, to, total};
                }
                i = j;
            }
            sh.n_segments = n;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the queries, for the products
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0), tS = tmem, tO = tmem + 2 * C_KEYS;
    const int total = __shfl_sync(0xffffffffu, sh.n_segments ? sh.segments[sh.n_segments - 1].tiles : 0, 0);
    const int first = (int)((long long)total * split / a.splits), last = (int)((long long)total * (split + 1) / a.splits), count = last - first;
    const auto begin_of = [&](int seg, int tile) { // first position of a tile of the list
        return sh.segments[seg].begin + (tile - (seg ? sh.segments[seg - 1].tiles : 0)) * C_KEYS;
    };

    if (warp >= C_SOFTMAX && warp < C_ISSUER) {
        // ===== pages -> operands: a pair of warps for every place that a tile of keys or of values has =====
        constexpr int PIECES = HS / 8, PART = C_KEYS / C_PAIR;
        const int place = (warp - C_SOFTMAX) / C_PAIR, part = (warp - C_SOFTMAX) % C_PAIR;
        const bool is_k = place < C_K;
        const int at = is_k ? place : place - C_K, step = is_k ? C_K : C_V;
        const char *pool = (const char *)(is_k ? a.pool.keys : a.pool.values);
        const uint32_t to = kv4::s32(is_k ? sK : sV) + at * c_tile_bytes(HS);
        const void *full = is_k ? &sh.k_full[at] : &sh.v_full[at], *free = is_k ? &sh.k_free[at] : &sh.v_free[at];
        int seg = 0;
        for (int j = at, turn = 0; j < count; j += step, turn++) {
            while (sh.segments[seg].tiles <= first + j) seg++;
            const int pos = begin_of(seg, first + j) + part * PART + lane, end = sh.segments[seg].end;
            const int *table = a.rows.table(sh.segments[seg].sequence);
            unsigned row[PART / 32];
#pragma unroll
            for (int h = 0; h < PART / 32; h++) row[h] = pos + 32 * h < end ? row_at(a.pool, table, pos + 32 * h, kvh) : NO_ROW;
            if (turn > 0 && !__all_sync(0xffffffffu, c_wait(free, (turn - 1) & 1, &sh.bail))) break; // keys: the scores of tile j - 3 stand; values: the products of tile j - 2 have read them
#pragma unroll
            for (int h = 0; h < PART / 32; h++) {
                const unsigned have = __ballot_sync(0xffffffffu, row[h] != NO_ROW);
                if (is_k && lane == 0) sh.have[at][part * (PART / 32) + h] = have;
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    const int n = lane + 32 * i, r = n / PIECES, p = n % PIECES;
                    const unsigned from = __shfl_sync(0xffffffffu, row[h], r);
                    cp16_or_zeros(from != NO_ROW, to + c_at<HS>(part * PART + 32 * h + r, p), pool + (from == NO_ROW ? 0 : ((size_t)from * HS + p * 8) * 2));
                }
            }
            cp_commit();
            cp_wait<0>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(full);
        }
    } else if (warp == C_ISSUER) {
        // ===== products =====
        constexpr uint32_t types = F16 ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = (1u << 4) | types | ((uint32_t)(C_KEYS >> 3) << 17) | ((uint32_t)(C_ROWS >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | types | (1u << 16) | ((uint32_t)(HS >> 3) << 17) | ((uint32_t)(C_ROWS >> 4) << 24); // bit 16: the second operand is entry-major
        const uint32_t q = kv4::s32(sQ), lead = lane == 0;
        const auto passed = [&](const void *bar, unsigned parity) { return __all_sync(0xffffffffu, c_wait<false>(bar, parity, &sh.bail)) != 0; };
        const auto scores = [&](int stage, int h) { // S = Q K^T
            const uint32_t k0 = kv4::s32(sK) + stage * c_tile_bytes(HS);
#pragma unroll
            for (int k = 0; k < HS / 16; k++) umma_ss(tS + h * C_KEYS, k_major<HS>(q, k), k_major<HS>(k0, k), idesc_s, k > 0, lead);
            umma_commit(&sh.s_full[h], lead);
        };
        unsigned turn = 0; // bit h: the phase of the stream's next probabilities
        bool ok = true;
        for (int j = 0; j < min(count, 2) && ok; j++) {
            if (!(ok = passed(&sh.k_full[j], 0))) break;
            fence_after();
            scores(j, j);
        }
        int stage = 0, ahead = 2; // of the keys of tiles j and j + 2
        unsigned phase = 0;
        for (int j = 0; j < count && ok; j++) {
            const int h = j & 1;
            volatile unsigned *again = &sh.again[h], *repeat = &sh.repeat[h];
            if (!(ok = passed(&sh.v_full[h], j >> 1 & 1))) break; // (first what is ready early)
            if (!(ok = passed(&sh.p_full[h], turn >> h & 1))) break;
            turn ^= 1u << h;
            if (__any_sync(0xffffffffu, *again != 0)) { // these probabilities do not count: the scores once more
                if (lead) {
                    *again = 0;
                    *repeat = 1;
                }
                __syncwarp();
                fence_after();
                scores(stage, h);
                if (!(ok = passed(&sh.p_full[h], turn >> h & 1))) break;
                turn ^= 1u << h;
            }
            if (lead) bar_arrive(&sh.k_free[stage]);
            fence_after();
            const uint32_t v0 = kv4::s32(sV) + h * c_tile_bytes(HS);
#pragma unroll
            for (int k = 0; k < C_KEYS / 16; k++) // O += P V
                umma_ts(tO + h * C_KEYS, tS + h * C_KEYS + (k / 4) * (C_KEYS / 2) + (k % 4) * 8, entry_major<HS>(v0, k), idesc_o, j > 1 || k > 0, lead);
            umma_commit(&sh.v_free[h], lead);
            if (lead) *repeat = 0;
            __syncwarp();
            if (j + 2 < count) {
                if (!(ok = passed(&sh.k_full[ahead], phase))) break;
                fence_after();
                scores(ahead, h);
            } else umma_commit(&sh.s_full[h], lead);
            if (++stage == C_K) stage = 0;
            if (++ahead == C_K) {
                ahead = 0;
                phase ^= 1;
            }
        }
        // what is under way ends before the tensor memory goes: the warps of the rows have waited for it, or one of them has given up
        unsigned none = 0;
        umma_commit(&sh.drained, lead);
        if (!c_wait(&sh.drained, 0, &none)) *reinterpret_cast<volatile unsigned *>(&sh.bail) = 1u;
    } else if (warp < C_SOFTMAX) {
        // ===== rows: two threads a stream, 64 positions of a tile a thread =====
        constexpr int PIECE = 16, COLUMNS = C_KEYS / 2;
        const int side = warp / 8, stream = warp / 4 % 2, r = tid % C_ROWS, token = token_of(r);
        const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16, row_s = tS + lanes + stream * C_KEYS + side * COLUMNS, row_o = tO + lanes + stream * C_KEYS;
        unsigned met = 0;
        int j = stream - 2; // the tile
        const auto meet = [&]() { // the two warps of a row; a wait with an end, as all here: one of them may have given up
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.pair[warp % 8]);
            return __all_sync(0xffffffffu, c_wait(&sh.pair[warp % 8], met++ & 1, &sh.bail)) != 0;
        };
        int lo = 0, hi = 0, own = -1, seg = 0;
        if (token < tokens && sh.segment[token] >= 0) {
            own = sh.segment[token];
            visible(sh.pos[token], a.window, lo, hi);
        }
        float top = -CUDART_INF_F, l = 0.0f, sum = 0.0f; // the row's largest product so far; of this thread's positions the sum, and that of a tile that may yet be repeated
        bool ok = true, fresh = false;
        float base = 0.0f, ref = -LIFT; // top where there is one, times the factor, and 2^LIFT below
        int from = 0, to = 0, next = 0; // the tile's positions [from, to) are seen, counted from this thread's first; the segment's end
        for (unsigned turn = 0; stream < count; turn++) {
            if (GIVE_UP && j + 2 >= count) {
                c_wait(&sh.pair[warp % 8], met & 1, &sh.bail);
                break;
            }
            ok = __all_sync(0xffffffffu, c_wait(&sh.s_full[stream], turn & 1, &sh.bail));
            if (!ok) break;
            fence_after();
            const bool repeat = *reinterpret_cast<volatile unsigned *>(&sh.repeat[stream]);
            if (!repeat) {
                l += sum;
                if ((j += 2) >= count) break;
                if (first + j >= next) {
                    while (sh.segments[seg].tiles <= first + j) seg++;
                    next = sh.segments[seg].tiles;
                    const int key0 = begin_of(seg, first + j) + side * COLUMNS;
                    from = own == seg ? lo - key0 : 0;
                    to = own == seg ? hi - key0 : 0;
                } else {
                    from -= 2 * C_KEYS;
                    to -= 2 * C_KEYS;
                }
                fresh = top == -CUDART_INF_F && max(from, -side * COLUMNS) < min(to, C_KEYS - side * COLUMNS); // the first that the row sees: no maximum yet
            }
            // bits of this thread's positions that its row sees, where not all do
            const unsigned have_lo = sh.have[j % C_K][2 * side], have_hi = sh.have[j % C_K][2 * side + 1];
            const auto bits = [](int from, int to) { // [from, to) of 32
                const unsigned below = to <= 0 ? 0u : to >= 32 ? 0xffffffffu : (1u << to) - 1u;
                return from <= 0 ? below : from >= 32 ? 0u : below & (0xffffffffu << from);
            };
            const unsigned seen_lo = bits(from, to) & have_lo, seen_hi = bits(from - 32, to - 32) & have_hi;
            const bool whole = (seen_lo & seen_hi) == 0xffffffffu;
            // One pass with the maximum as it stands.  It moves rarely, and a sum of more than 2^8 shows that it has to: the probabilities, which have taken the place of the scores, are
            // dropped, the scores come once more, and the tile's maximum is looked for first.  (A maximum of every tile in front of the exponentials would read the scores twice.)
            const bool special = __any_sync(0xffffffffu, repeat || fresh || !whole || !(fabsf(ref) <= 65536.0f));
            if (special && __any_sync(0xffffffffu, repeat || fresh)) { // (the same for both warps of a row)
                float mx = -CUDART_INF_F;
#pragma unroll 1
                for (int q = 0; q < COLUMNS; q += PIECE) {
                    uint32_t x[PIECE];
                    tmem_ld16(row_s + q, x);
                    const unsigned seen = (q < 32 ? seen_lo : seen_hi) >> q % 32;
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < PIECE; i++) mx = fmaxf(mx, seen & (1u << i) ? __uint_as_float(x[i]) : -CUDART_INF_F);
                }
                sh.half_row[stream][side][r] = mx;
                ok = meet();
                if (!ok) break;
                mx = fmaxf(mx, sh.half_row[stream][side ^ 1][r]);
                const float grown = fmaxf(top, mx), alpha = top == grown ? 1.0f : ex2((top - grown) * factor);
                top = grown;
                l *= alpha;
                if (j > 1 && __any_sync(0xffffffffu, alpha != 1.0f)) { // (the product of tile j - 2 came before these scores)
#pragma unroll 1
                    for (int q = side * HS / 2; q < (side + 1) * HS / 2; q += PIECE) {
                        uint32_t o[PIECE];
                        tmem_ld16(row_o + q, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < PIECE; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st16(row_o + q, o);
                    }
                }
                base = top == -CUDART_INF_F ? 0.0f : top;
                ref = base * factor - LIFT;
            }
            // P takes the place of S: piece q of 16 scores is read before its 8 columns are written, [8 q, 8 q + 8)
            if (special && !__any_sync(0xffffffffu, (seen_lo | seen_hi) != 0u)) { // other rows' tile
                const uint32_t p[PIECE / 2] = {};
                sum = 0.0f;
#pragma unroll 1
                for (int q = 0; q < COLUMNS / 2; q += PIECE / 2) tmem_st8(row_s + q, p);
            } else if (special && __any_sync(0xffffffffu, !whole || !(fabsf(ref) <= 65536.0f))) { // a border, or scores so large that their products and the maximum's round apart
                sum = 0.0f;
#pragma unroll 1
                for (int q = 0; q < COLUMNS; q += PIECE) {
                    uint32_t x[PIECE], p[PIECE / 2];
                    tmem_ld16(row_s + q, x);
                    const unsigned seen = (q < 32 ? seen_lo : seen_hi) >> q % 32;
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < PIECE; i++) {
                        const float e = seen & (1u << i) ? ex2(fmaf(__uint_as_float(x[i]) - base, factor, LIFT)) : 0.0f;
                        sum += e;
                        x[i] = __float_as_uint(e);
                    }
#pragma unroll
                    for (int i = 0; i < PIECE / 2; i++) p[i] = pack2<T>(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
                    tmem_st8(row_s + q / 2, p);
                }
            } else {
                const unsigned long long factor2 = pack_f32x2(factor, factor), ref2 = pack_f32x2(-ref, -ref);
                unsigned long long part[2] = {0ull, 0ull};
                uint32_t s[2][PIECE];
                tmem_ld16(row_s, s[0]);
#pragma unroll
                for (int q = 0; q < COLUMNS / PIECE; q++) {
                    uint32_t(&x)[PIECE] = s[q & 1];
                    tmem_ld_wait();
                    if (q + 1 < COLUMNS / PIECE) tmem_ld16(row_s + (q + 1) * PIECE, s[q + 1 & 1]);
                    uint32_t p[PIECE / 2];
#pragma unroll
                    for (int i = 0; i < PIECE / 2; i++) {
                        float e0, e1;
                        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), factor2, ref2), e0, e1);
                        e0 = ex2(e0);
                        e1 = ex2(e1);
                        part[i & 1] = add_f32x2(part[i & 1], pack_f32x2(e0, e1));
                        p[i] = pack2<T>(e0, e1);
                    }
                    tmem_st8(row_s + q * (PIECE / 2), p);
                }
                float a0, a1, b0, b1;
                unpack_f32x2(part[0], a0, a1);
                unpack_f32x2(part[1], b0, b1);
                sum = (a0 + a1) + (b0 + b1);
            }
            const bool over = __any_sync(0xffffffffu, !repeat && sum > TOO_MUCH);
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (over) *reinterpret_cast<volatile unsigned *>(&sh.again[stream]) = 1u;
                bar_arrive(&sh.p_full[stream]);
            }
        }
        sh.half_row[stream][side][r] = l;
        sh.top[stream][r] = top;
        fence_before();
    }
    __syncthreads();
    // ===== results: the streams are joined; a warp takes 32 rows and 32 entries =====
    const bool gave_up = sh.bail != 0u;
    const auto put16 = [&](float v) { return a.out_type == B200_GGML_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v)); };
    float2 *stats = reinterpret_cast<float2 *>(a.work + (size_t)a.rows.n * a.heads * a.splits * HS);
    if (warp < 4 * (HS / 32)) {
        fence_after();
        const int q = warp / 4, r = warp % 4 * 32 + lane, token = token_of(r), row = token0 + token, head = kvh * mul + r - token * mul;
        const bool on = token < tokens && sh.seq[min(token, C_ROWS - 1)] >= 0;
        const float t0 = sh.top[0][r], t1 = sh.top[1][r], top = fmaxf(t0, t1), base = top == -CUDART_INF_F ? 0.0f : top;
        const float a0 = t0 == base ? 1.0f : ex2((t0 - base) * factor), a1 = t1 == base ? 1.0f : ex2((t1 - base) * factor);
        float l = a0 * (sh.half_row[0][0][r] + sh.half_row[0][1][r]) + a1 * (sh.half_row[1][0][r] + sh.half_row[1][1][r]);
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; i++) o[i] = 0.0f;
        if (!gave_up)
            for (int h = 0; h < min(count, 2); h++) { // (a stream without tiles has no sums)
#pragma unroll
                for (int i = 0; i < 32; i += 16) {
                    uint32_t x[16];
                    tmem_ld16(tO + ((uint32_t)(warp % 4 * 32) << 16) + h * C_KEYS + q * 32 + i, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int u = 0; u < 16; u++) o[i + u] = fmaf(h ? a1 : a0, __uint_as_float(x[u]), o[i + u]);
                }
            }
        else l = CUDART_NAN_F;
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 32; i++) finite &= fabsf(o[i]) < CUDART_INF_F;
        if (on && !finite) atomicOr(&sh.bad[r / 32], 1u << (r % 32));
        fence_before();
        if (a.splits > 1) {
            if (on) {
                const size_t part = ((size_t)row * a.heads + head) * a.splits + split;
                if (q == 0) stats[part] = make_float2(top * factor - LIFT, l);
                float4 *w = reinterpret_cast<float4 *>(a.work + part * HS + q * 32);
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
        } else if (on) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = gave_up ? 0x7fff7fffu : put16(o[2 * i] * inv) | (uint32_t)put16(o[2 * i + 1] * inv) << 16;
            uint16_t *out = (uint16_t *)a.out + row * a.ldo + (size_t)head * HS + q * 32;
            if (a.vec_out)
#pragma unroll
                for (int i = 0; i < 4; i++) reinterpret_cast<uint4 *>(out)[i] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
            else
#pragma unroll
                for (int i = 0; i < 32; i++) out[i] = (uint16_t)(y[i / 2] >> (i & 1) * 16);
        }
    }
    __syncthreads();
    if (warp == C_SOFTMAX) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (gave_up || (sh.bad[0] | sh.bad[1] | sh.bad[2] | sh.bad[3]) == 0u) return;
    // ===== rows whose sums are not finite: once more, one after the other, 2^-40 below their maximum =====
    constexpr int AT_ONCE = 4096, LANES = HS / 2, GROUPS = C_THREADS / LANES;
    float *p = reinterpret_cast<float *>(sK);
    float2 *sums = reinterpret_cast<float2 *>(sV); // [group][pair of entries]
    for (int r = 0; r < C_ROWS; r++) {
        if (!(sh.bad[r / 32] >> (r % 32) & 1u)) continue;
        const int token = token_of(r), row = token0 + token, head = kvh * mul + r - token * mul, seg = sh.segment[token];
        int lo = 0, hi = 0;
        if (seg >= 0) { // what this CTA's tiles hold of it
            visible(sh.pos[token], a.window, lo, hi);
            const int before = seg ? sh.segments[seg - 1].tiles : 0, b = max(first, before) - before, e = min(last, sh.segments[seg].tiles) - before;
            lo = max(lo, sh.segments[seg].begin + b * C_KEYS);
            hi = min(hi, sh.segments[seg].begin + e * C_KEYS);
        }
        float top = -CUDART_INF_F, l = 0.0f;
        float2 o = make_float2(0.0f, 0.0f);
        const int pair = tid % LANES, group = tid / LANES;
        for (int k0 = lo; k0 < hi; k0 += AT_ONCE) {
            const int n = min(AT_ONCE, hi - k0);
            const int *table = a.rows.table(sh.segments[seg].sequence);
            float mx = -CUDART_INF_F;
            __syncthreads();
            for (int i = tid; i < n; i += C_THREADS) {
                const unsigned at = row_at(a.pool, table, k0 + i, kvh);
                float s = CUDART_NAN_F;
                if (at != NO_ROW) {
                    const uint4 *k = reinterpret_cast<const uint4 *>((const T *)a.pool.keys + (size_t)at * HS);
                    s = 0.0f;
                    for (int c = 0; c < HS / 8; c++) {
                        const uint4 x = k[c], q = *reinterpret_cast<const uint4 *>(sQ + c_at<HS>(r, c));
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const float2 x2 = unpack2<T>(xs[u]), q2 = unpack2<T>(qs[u]);
                            s = fmaf(x2.x, q2.x, s);
                            s = fmaf(x2.y, q2.y, s);
                        }
                    }
                    mx = fmaxf(mx, s);
                }
                p[i] = s;
            }
            const float grown = fmaxf(top, block_all(sh, mx, false)), base = grown == -CUDART_INF_F ? 0.0f : grown, alpha = top == grown ? 1.0f : ex2((top - base) * factor);
            top = grown;
            float part = 0.0f;
            for (int i = tid; i < n; i += C_THREADS) {
                const bool page = row_at(a.pool, table, k0 + i, kvh) != NO_ROW;
                const float e = page ? ex2(fmaf(p[i] - base, factor, -40.0f)) : 0.0f;
                p[i] = page ? e : -1.0f; // (-1: nobody sees it)
                part += e;
            }
            l = l * alpha + block_all(sh, part, true);
            o.x *= alpha;
            o.y *= alpha;
            if (group < GROUPS)
                for (int i = group; i < n; i += GROUPS) {
                    const float e = p[i];
                    if (e == -1.0f) continue;
                    const float2 v = unpack2<T>(reinterpret_cast<const uint32_t *>((const T *)a.pool.values + (size_t)row_at(a.pool, table, k0 + i, kvh) * HS)[pair]);
                    o.x = fmaf(e, v.x, o.x);
                    o.y = fmaf(e, v.y, o.y);
                }
        }
        __syncthreads();
        if (group < GROUPS) sums[tid] = o;
        __syncthreads();
        if (tid < LANES) {
            for (int i = 1; i < GROUPS; i++) {
                const float2 x = sums[i * LANES + tid];
                o.x += x.x;
                o.y += x.y;
            }
            if (a.splits > 1) {
                const size_t part = ((size_t)row * a.heads + head) * a.splits + split;
                if (tid == 0) stats[part] = make_float2(top * factor + 40.0f, l);
                reinterpret_cast<float2 *>(a.work + part * HS)[tid] = make_float2(o.x, o.y);
            } else {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                uint16_t *out = (uint16_t *)a.out + row * a.ldo + (size_t)head * HS + 2 * tid;
                out[0] = put16(o.x * inv);
                out[1] = put16(o.y * inv);
            }
        }
    }
}

} // namespace paged
