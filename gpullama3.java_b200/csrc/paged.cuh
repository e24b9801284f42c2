// paged.cuh -- a 16-bit key/value cache in pages: append (head norms, rotation and rounding in one pass) and the attention of rows over the pages of their sequences.
//
// The pool is [page][key/value head][position of the page][entry], keys and values apart, FP16 or BF16; position p of a sequence lies in page table[p >> shift], row p & (2^shift - 1).
// So the rows of a page and head are one contiguous stretch, and a row is named by one 32-bit number, (page * heads + head) * page_size + row.  A table entry outside the pool is no
// page: nothing is stored there, and its positions are seen by nobody.
#pragma once
#include "kv4.cuh"

namespace paged {

using kv4::bf16;
using kv4::cp16;
using kv4::cp_commit;
using kv4::cp_wait;
using kv4::ex2;
using kv4::load8;
using kv4::put;
using kv4::visible;

constexpr unsigned NO_ROW = 0xffffffffu;

struct Pool {
    void *keys, *values;
    int pages, kv_heads, shift; // positions of a page: 2^shift
};
struct Rows { // row r stands at position positions[r] of sequence `sequences ? sequences[r] : 0`
    const int *positions, *sequences, *tables;
    long long ld_table;
    int n, n_sequences, context; // context: positions that a table names
    __device__ __forceinline__ int sequence_of(int r) const { return sequences ? sequences[r] : 0; }
    // its sequence, or -1 for a padding row
    __device__ __forceinline__ int place(int r, int &pos) const {
        const int s = sequence_of(r);
        pos = positions[r];
        return s < 0 || s >= n_sequences || pos >= context ? -1 : s;
    }
    __device__ __forceinline__ const int *table(int s) const { return tables + s * ld_table; }
};
// The number of a head's row at a position, or NO_ROW.
__device__ __forceinline__ unsigned row_at(const Pool &p, const int *table, int pos, int head) {
    const int page = table[pos >> p.shift];
    return (unsigned)page < (unsigned)p.pages ? (((unsigned)page * p.kv_heads + head) << p.shift) + (pos & ((1 << p.shift) - 1)) : NO_ROW;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return kv4::pack_f16(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<bf16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w) { return kv4::to_f32x2(w, (const T *)nullptr); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }

// ---- append ---------------------------------------------------------------------------------------------------------------------------------------------------
struct Append {
    Pool pool;
    Rows rows;
    const void *q, *k, *v;
    long long ldq, ldk, ldv, ldo; // entries between rows
    int heads;                    // query heads; 0: none
    int interleaved, turned;      // turned: entries of a head that are rotated, its first ones
    int vec, vec_out, vec_tables; // rows, query results and the rotation's rows start on 16-byte boundaries
    const float *q_norm, *k_norm, *cos, *sin;
    float eps;
    void *q_out;
};

// A CTA takes a row, or some of its heads.  Lanes of a head: 8 entries each; WIDTH lanes (a power of two) serve one head.  Mean of squares in 64 bits (FP32 squares leave FP32's range from 2^64 on).  Pairs of neighbours lie in a
// lane; pairs half the rotated part apart lie in lanes a fixed distance apart where half of it is a multiple of 8, and are read once more from memory where it is not.
// Bytes are its floor: 512 rows of (32 + 2 * 8) heads of 128 in BF16 read and write 12.8 MB, 2.0 us; in a captured graph it takes 7.4 (8.2 as a call), a step's row 2.4: latency, a chain of loads (position, then
// page and angles) and 64-bit sums; a warp's index by division of a flat one was 1.2 us more.
template <int HS, typename T, typename C> __global__ void __launch_bounds__(256) k_paged_append(const Append a) {
    constexpr int L = HS / 8, WIDTH = L <= 4 ? 4 : L <= 8 ? 8 : L <= 16 ? 16 : 32, PER_WARP = 32 / WIDTH;
    const int lane = threadIdx.x & 31, li = lane & (WIDTH - 1), G = a.pool.kv_heads, total = a.heads + 2 * G;
    const int row = blockIdx.x, which = (blockIdx.y * 8 + (threadIdx.x >> 5)) * PER_WARP + lane / WIDTH;
    const bool is_q = which < a.heads, is_v = which >= a.heads + G, there = which < total && li < L;
    const int head = is_q ? which : is_v ? which - a.heads - G : which - a.heads, e = li * 8;
    const T *src = (is_q ? (const T *)a.q + (long long)row * a.ldq : is_v ? (const T *)a.v + (long long)row * a.ldv : (const T *)a.k + (long long)row * a.ldk) + (size_t)head * HS;
    float x[8]; // (on its way while its place is looked up)
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    if (there) load8(src + e, x, a.vec);
    int pos = -1;
    const int seq = a.rows.place(row, pos);
    if (seq < 0 || pos < 0) return; // (the whole CTA)
    const bool mine = there;
    const unsigned at = mine && !is_q ? row_at(a.pool, a.rows.table(seq), pos, head) : NO_ROW;
    const float *norm = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    float s = 1.0f;
    if (a.q_norm || a.k_norm) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
        for (int o = WIDTH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (norm && mine) {
            s = (float)rsqrt(ss * (1.0 / HS) + (double)a.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = norm[e + i] * (s * x[i]);
        }
    }
    if (a.cos) {
        const int half = a.turned / 2;
        const float *cs = a.cos + (size_t)pos * half, *sn = a.sin + (size_t)pos * half;
        const bool turns = mine && !is_v && e < a.turned;
        if (a.interleaved) {
            if (turns) {
                float c[4], n[4];
                if (a.vec_tables) {
                    const float4 u = *reinterpret_cast<const float4 *>(cs + e / 2), w = *reinterpret_cast<const float4 *>(sn + e / 2);
                    c[0] = u.x; c[1] = u.y; c[2] = u.z; c[3] = u.w;
                    n[0] = w.x; n[1] = w.y; n[2] = w.z; n[3] = w.w;
                } else
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool in = e + 2 * i < a.turned;
                        c[i] = in ? cs[e / 2 + i] : 1.0f;
                        n[i] = in ? sn[e / 2 + i] : 0.0f;
                    }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float u = x[2 * i], w = x[2 * i + 1];
                    if (e + 2 * i >= a.turned) break;
                    x[2 * i] = u * c[i] - w * n[i];
                    x[2 * i + 1] = u * n[i] + w * c[i];
                }
            }
        } else if (half % 8 == 0) {
            const bool low = e < half;
            const int partner = lane - li + (e < a.turned ? low ? li + half / 8 : li - half / 8 : li);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], partner);
            if (turns) {
                float c[8], n[8];
                load8(cs + (low ? e : e - half), c, a.vec_tables);
                load8(sn + (low ? e : e - half), n, a.vec_tables);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = low ? x[i] * c[i] - y[i] * n[i] : y[i] * n[i] + x[i] * c[i];
            }
        } else if (turns) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = e + i;
                if (j >= a.turned) break;
                const bool low = j < half;
                const int other = low ? j + half : j - half;
                float y = to_f32(src[other]);
                if (norm) y = norm[other] * (s * y);
                const float c = cs[low ? j : j - half], n = sn[low ? j : j - half];
                x[i] = low ? x[i] * c - y * n : y * n + x[i] * c;
            }
        }
    }
    if (!mine || (!is_q && at == NO_ROW)) return;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = pack2<C>(x[2 * i], x[2 * i + 1]);
    if (!is_q) *reinterpret_cast<uint4 *>((C *)(is_v ? a.pool.values : a.pool.keys) + (size_t)at * HS + e) = make_uint4(w[0], w[1], w[2], w[3]);
    else {
        uint16_t *o = (uint16_t *)a.q_out + (long long)row * a.ldo + (size_t)head * HS + e;
        if (a.vec_out) *reinterpret_cast<uint4 *>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = (uint16_t)(w[i / 2] >> 16 * (i & 1));
    }
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------------------------------
struct Step {
    Pool pool;
    Rows rows;
    const void *q; // of the cache's type
    long long ldq, ldo;
    int heads, window, vec, vec_out, out_type;
    float scale;
    void *out;
    int mul, of;                       // query heads of a key/value head; r / mul = r of >> 16 for the rows of a unit of several tokens
    int tokens, blocks; // rows of a group are `tokens` neighbouring ones; a unit is one of its `blocks` blocks of one key/value head
    int ctas;           // that find room on the GPU, where units are shared out (0: a CTA a unit)
    int splits;         // (chunks) CTAs of a unit
    float *work;        // parts of units that several CTAs share.  ctas: [CTA][row] entries, behind them reference and sum; splits: [row][head][split] likewise
};

constexpr int STEP_WARPS = 2, STEP_GROUPS = 256; // warps of a CTA; units of tokens that it shares out by their lengths
constexpr int STEP_SHARED_ROWS = 4 * STEP_GROUPS; // rows of all groups, then
__host__ __device__ constexpr int step_keys(int hs) { return hs == 256 ? 16 : 32; }           // positions that a warp takes at a time: a tile
__host__ __device__ constexpr int step_stages(int hs) { return hs == 32 || hs == 256 ? 3 : 2; } // tiles that it has room for
__host__ __device__ constexpr int step_stage_bytes(int hs) { return step_keys(hs) * hs * 4; } // keys and values
__host__ __device__ constexpr int step_rows(int nr) { return 8 * nr; }
__host__ __device__ constexpr int step_tokens_most() { return 32; }
__host__ __device__ constexpr int part_stride(int hs) { return hs + 4; } // (rows 8 banks apart two by two)
__host__ __device__ constexpr size_t step_smem_bytes(int hs, int nr) {
    const size_t ring = (size_t)STEP_WARPS * step_stages(hs) * step_stage_bytes(hs), parts = (size_t)STEP_WARPS * step_rows(nr) * part_stride(hs) * 4;
    return (ring > parts ? ring : parts) + (size_t)step_rows(nr) * hs * 2;
}
__host__ __device__ constexpr int step_ctas(int hs, int nr) { // of an SM, as far as its shared memory and registers go
    const int n = (int)(233472 / (step_smem_bytes(hs, nr) + 3 * 1024)), most = hs <= 64 && nr >= 3 ? 4 : 8;
    return n < 1 ? 1 : n > most ? most : n;
}

__device__ __forceinline__ uint32_t s32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T> __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { kv4::mma_f16(d, a, b0, b1); }
template <> __device__ __forceinline__ void mma<bf16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
using kv4::transpose8x8;
__device__ __forceinline__ void cp16_or_zeros(bool on, uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// 16-byte piece c of row r of a tile whose rows are HS entries: eight neighbouring rows of a piece lie in different banks.
template <int HS> __device__ __forceinline__ int turn_of(int r) { return HS % 64 == 0 ? r & 7 : r >> 1 & 3; }
template <int HS> __device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)(r * HS * 2 + ((c ^ turn_of<HS>(r)) << 4)); }

struct Segment { // a run of tokens of one sequence: tiles [begin, end) of its positions [lo, hi), those that any of them sees; tiles of all segments up to and with this one
    int sequence, begin, end, lo, hi, tiles;
};

__device__ __forceinline__ void put_results(const Step &a, int row, int head, int hs, int e, float4 o) { // entries e .. e + 3 of a row's head
    const long long at = row * a.ldo + (long long)head * hs + e;
    const float x[4] = {o.x, o.y, o.z, o.w};
    if (a.out_type == B200_GGML_F32) {
        float *p = (float *)a.out + at;
        if (a.vec_out) *reinterpret_cast<float4 *>(p) = o;
        else
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = x[i];
    } else {
        const uint2 w = a.out_type == B200_GGML_F16 ? make_uint2(pack2<__half>(o.x, o.y), pack2<__half>(o.z, o.w)) : make_uint2(pack2<bf16>(o.x, o.y), pack2<bf16>(o.z, o.w));
        uint16_t *p = (uint16_t *)a.out + at;
        if (a.vec_out) *reinterpret_cast<uint2 *>(p) = w;
        else {
            p[0] = (uint16_t)w.x; p[1] = (uint16_t)(w.x >> 16);
            p[2] = (uint16_t)w.y; p[3] = (uint16_t)(w.y >> 16);
        }
    }
}

// The segments of a group of tokens, in order: emit(first token, last token + 1, segment), sequence -1 for a run that sees nothing.
template <typename P, typename F> __device__ __forceinline__ void segments_of_group(const Step &a, int tokens, int KT, P place, F emit) {
    int total = 0;
    for (int i = 0; i < tokens;) {
        int pos;
        const int s = place(i, pos);
        int j = i, from = INT_MAX, to = 0;
        for (int sj = s; sj == s;) {
            int lo, hi;
            visible(max(pos, -1), a.window, lo, hi);
            if (hi > lo) { from = min(from, lo); to = max(to, hi); }
            if (++j == tokens) break;
            sj = place(j, pos);
        }
        Segment sg = {-1, 0, 0, 0, 0, total};
        if (s >= 0 && to > 0) {
            sg = {s, from / KT, (to - 1) / KT + 1, from, to, 0};
            total += sg.end - sg.begin;
            sg.tiles = total;
        }
        emit(i, j, sg);
        i = j;
    }
}
// How units are shared out over CTAs, by what their rows see: with S tiles a CTA at most, a unit of t tiles gets n = ceil(t / S) CTAs, even shares.  S is the smallest, to a sixteenth, with which
// all CTAs find room on the GPU at once (where there are many units: an even share of all tiles).  Every CTA finds its own place: all of them look at the rows' positions.
constexpr int SHARE_LEAST = 8; // tiles of a CTA, where a unit has so many
struct Shares {
    int before[STEP_GROUPS + 1]; // CTAs of the groups in front
    int tiles[STEP_GROUPS];      // of a group, for one head and block
    int2 at[STEP_GROUPS];        // LONE: its sequence and position
    long long sums[8];
};
template <int THREADS> __device__ __forceinline__ long long block_sum(long long v, long long *sums) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = v;
    __syncthreads();
    v = sums[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; w++) v += sums[w];
    return v;
}
static_assert(STEP_SHARED_ROWS * 8 + sizeof(Shares) <= (size_t)STEP_WARPS * step_stages(32) * step_stage_bytes(32), "the smallest ring holds what is needed before it");
// The whole CTA; stage: room for the rows' sequences and positions, where groups have several of them.
template <int KT, bool LONE, int THREADS> __device__ __forceinline__ void share_out(const Step &a, Shares &sh, int2 *stage) {
    constexpr int PER = STEP_GROUPS / THREADS;
    const int tid = threadIdx.x, lane = tid & 31, groups = (a.rows.n + a.tokens - 1) / a.tokens, per_group = a.pool.kv_heads * a.blocks;
    if constexpr (LONE) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int g = tid + i * THREADS;
            int pos = -1, lo, hi, s = -1;
            if (g < groups) s = a.rows.place(g, pos);
            pos = max(pos, -1);
            visible(pos, a.window, lo, hi);
            sh.at[g] = make_int2(s, pos);
            sh.tiles[g] = s >= 0 && hi > lo ? (hi - 1) / KT + 1 - lo / KT : 0;
        }
    } else {
#pragma unroll 4
        for (int r = tid; r < a.rows.n; r += THREADS) {
            int pos;
            const int s = a.rows.place(r, pos);
            stage[r] = make_int2(s, pos);
        }
        __syncthreads();
        for (int g = tid; g < STEP_GROUPS; g += THREADS) {
            int tiles = 0;
            const int token0 = g * a.tokens;
            if (g < groups)
                segments_of_group(a, min(a.tokens, a.rows.n - token0), KT, [&](int t, int &pos) { pos = stage[token0 + t].y; return stage[token0 + t].x; },
                                  [&](int, int, const Segment &sg) { tiles = sg.tiles; });
            sh.tiles[g] = tiles;
        }
    }
    __syncthreads();
    int mine[PER];
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        mine[i] = sh.tiles[tid * PER + i];
        sum += mine[i];
    }
    const long long total = block_sum<THREADS>(sum, sh.sums) * per_group;
    int share = (int)min(max((total + a.ctas - 1) / a.ctas, (long long)SHARE_LEAST), 1LL << 30);
    if (groups * per_group <= a.ctas / 4 * 3)
        for (;;) { // (at most a few dozen times: the units alone take three quarters of the room)
            long long ctas = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) ctas += (mine[i] + share - 1) / share;
            if (block_sum<THREADS>(ctas, sh.sums) * per_group <= a.ctas) break;
            share += max(1, share / 16);
        }
    int ctas = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int n = (mine[i] + share - 1) / share * per_group;
        mine[i] = ctas;
        ctas += n;
    }
    int run = ctas;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += x;
    }
    __syncthreads();
    if (lane == 31) sh.sums[tid / 32] = run;
    __syncthreads();
    run -= ctas;
    for (int w = 0; w < tid / 32; w++) run += (int)sh.sums[w];
#pragma unroll
    for (int i = 0; i < PER; i++) sh.before[tid * PER + i] = run + mine[i];
    if (tid == THREADS - 1) sh.before[STEP_GROUPS] = run + ctas;
    __syncthreads();
}

// Rows (tokens x query heads of one key/value head) in blocks of 8 NR; LONE: of a single token, all on the same positions.  A CTA takes a unit, or an even
// share of its tiles (Shares), and deals them to its warps in turn; each warp has a cp.async ring and a running reference of its own, and no barrier in the loop.  Parts
// are joined in shared memory, those of several CTAs through the workspace (k_paged_join_shares).  Nothing depends on an order of arrival.
//   scores  S[16 positions x 8 rows] = K Q^T, the cache's type, exact products, FP32 sums;  p = 2^(factor s - ref), factor = |scale| log2(e), the scale's sign is the queries'
//   values  O[16 entries x 8 rows] += V^T P with p in the cache's type, half a step off, as the result will be; with FP32 results as PARTS numbers, each what the ones before left: two of FP16
//           (22 bits), three of BF16 (24: two, 16 bits, put FP32 results three times as far off as FP32 sums are)
// (Rows as the products' eight columns: four query heads of a key/value head, the usual number, leave half of them empty, as rows they would leave three quarters, with twice the registers.)
// ref follows the largest score seen so far only when that passes it by more than 2^8 (the first does), so that few tiles have anything to rescale; with FP16 it lies 2^7 below, so that
// p reaches down to 2^-24 of 2^-15: a long tail of small ones still counts.
// A value that is infinite or NaN would reach every row of the block as 0 * NaN, also those that do not see it, and sums of large BF16 values may leave FP32's range before they are divided: a
// warp whose sums are not finite computes its share once more at the end, a row after the other in FP32, from what each sees, with BF16 2^-40 below its maximum (slow_rows).
// Bytes are its floor.  One row of 8 key/value heads of 128 over 131071 positions, 537 MB: 84-85 us (6.3 TB/s; floor 83), with the join 88 in a graph; 48 rows of up to 4099 positions of 8 heads of 64, 206 MB: 45
// (floor 32), with the join 47; 16 sequences of 5 drafted tokens, 20 rows, over up to 8191 positions, 285 MB: 62 (floor 44), with the join 67, where the chains of products of six warps an SM (tensor pipes 22 %)
// keep the copies from running ahead.  What a CTA holds was measured on these three: two warps with two tiles of 32 positions each; tiles of 16 with three places: 91, 47, 61-66; four warps: 90, 53-56, 62; products with
// positions as columns (16 rows at least): 90, 46, 86.  An even share of all tiles for every CTA, whichever units they are of, was slower (88, 53, 72): a second unit costs a CTA another 5 us.
template <int HS, typename T> __device__ __noinline__ void slow_rows(const Step &a, const unsigned char *sQ, int rows, int row0, int token0, int kvh, int first, int last, int warp, const Segment *segments, const int *segment_of,
                                                                     const int *pos_of, float factor, float *parts, float *wref, float *wsum) {
    constexpr int KT = step_keys(HS), E = HS / 32; // entries of a lane
    constexpr float DOWN = std::is_same<T, __half>::value ? 0.0f : 40.0f; // (sums of FP16 values stay in FP32's range as they are)
    const int lane = threadIdx.x & 31;
    for (int r = 0; r < rows; r++) {
        const int token = (row0 + r) / a.mul, own = segment_of[token];
        int lo, hi, seg = 0;
        visible(pos_of[token], a.window, lo, hi);
        float top = -CUDART_INF_F, l = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        for (int tile = first + warp; tile < last && own >= 0; tile += STEP_WARPS) {
            while (segments[seg].tiles <= tile) seg++;
            if (seg != own) continue;
            const int pos = (segments[seg].end - (segments[seg].tiles - tile)) * KT + lane;
            const unsigned at = lane < KT && pos >= lo && pos < hi ? row_at(a.pool, a.rows.table(segments[seg].sequence), pos, kvh) : NO_ROW;
            float s = -CUDART_INF_F;
            if (at != NO_ROW) {
                s = 0.0f;
                for (int c = 0; c < HS / 8; c++) {
                    const uint4 x = reinterpret_cast<const uint4 *>((const T *)a.pool.keys + (size_t)at * HS)[c], q = *reinterpret_cast<const uint4 *>(sQ + piece<HS>(r, c));
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const float2 x2 = unpack2<T>(xs[u]), q2 = unpack2<T>(qs[u]);
                        s = fmaf(x2.x, q2.x, s);
                        s = fmaf(x2.y, q2.y, s);
                    }
                }
            }
            const float grown = fmaxf(top, warp_max_f(s)), base = grown == -CUDART_INF_F ? 0.0f : grown, alpha = top == grown ? 1.0f : ex2((top - base) * factor);
            top = grown;
            const float p = at != NO_ROW ? ex2(fmaf(s - base, factor, -DOWN)) : 0.0f;
            l = l * alpha + p;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] *= alpha;
            const unsigned seen = __ballot_sync(0xffffffffu, at != NO_ROW);
            for (int k = 0; k < KT; k++) {
                const float w = __shfl_sync(0xffffffffu, p, k);
                const unsigned from = __shfl_sync(0xffffffffu, at, k);
                if (!(seen >> k & 1u)) continue;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = fmaf(w, to_f32(((const T *)a.pool.values + (size_t)from * HS)[e * 32 + lane]), o[e]);
            }
        }
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
#pragma unroll
        for (int e = 0; e < E; e++) parts[r * part_stride(HS) + e * 32 + lane] = o[e];
        if (lane == 0) {
            wref[r] = top * factor + DOWN;
            wsum[r] = l;
        }
    }
}

// CTAs of the grid where units are shared out; in the workspace, behind the parts' entries and statistics: Shares::before.
__host__ __device__ inline size_t shared_grid(const Step &a, int groups) { return (size_t)a.ctas + (size_t)groups * a.pool.kv_heads * a.blocks; }
template <int HS, int NR> __device__ __forceinline__ float2 *stats_of(const Step &a, int groups) { return reinterpret_cast<float2 *>(a.work + shared_grid(a, groups) * step_rows(NR) * HS); }
template <int HS, int NR> __device__ __forceinline__ int *plan_of(const Step &a, int groups) { return reinterpret_cast<int *>(stats_of<HS, NR>(a, groups) + shared_grid(a, groups) * step_rows(NR)); }

template <int HS, typename T, int NR, int PARTS, bool LONE> __global__ void __launch_bounds__(STEP_WARPS * 32, step_ctas(HS, NR)) k_paged_step(const Step a) {
    constexpr int KT = step_keys(HS), KB = KT / 16, S = step_stages(HS), ROWS = step_rows(NR), PIECES = HS / 8, STAGE = step_stage_bytes(HS), TOKENS = LONE ? 1 : step_tokens_most(), RB = HS * 2;
    constexpr bool F16 = std::is_same<T, __half>::value, QREG = HS * NR <= 256;
    constexpr float LIFT = F16 ? 7.0f : 0.0f;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Segment segments[TOKENS];
    __shared__ int seq_of[TOKENS], pos_of[TOKENS], segment_of[TOKENS], n_segments;
    __shared__ unsigned there[STEP_WARPS][S]; // positions of a tile that have a page
    __shared__ float wref[STEP_WARPS][ROWS], wsum[STEP_WARPS][ROWS], weight[STEP_WARPS][ROWS];
    unsigned char *sQ = smem + step_smem_bytes(HS, NR) - ROWS * RB;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    Shares &shares = *reinterpret_cast<Shares *>(smem + STEP_SHARED_ROWS * 8); // (where the rings will be)
    const int mul = a.mul, groups = (a.rows.n + a.tokens - 1) / a.tokens, per_group = a.pool.kv_heads * a.blocks;
    pdl_launch_dependents();
    int unit = blockIdx.x / per_group, within = blockIdx.x % per_group, part = 0, n_parts = 1;
    int2 sequence_position;
    if (a.ctas) {
        share_out<KT, LONE, STEP_WARPS * 32>(a, shares, reinterpret_cast<int2 *>(smem));
        if (blockIdx.x == 0) // for the join
            for (int i = tid; i <= groups; i += STEP_WARPS * 32) plan_of<HS, NR>(a, groups)[i] = shares.before[i];
        if ((int)blockIdx.x >= shares.before[groups]) return;
        int low = 0, high = groups - 1; // the last group that starts with this CTA or in front of it
        while (low < high) {
            const int mid = (low + high + 1) / 2;
            if (shares.before[mid] <= (int)blockIdx.x) low = mid;
            else high = mid - 1;
        }
        unit = low;
        n_parts = (shares.before[low + 1] - shares.before[low]) / per_group;
        const int at = blockIdx.x - shares.before[low];
        within = at % per_group; // (CTAs that run side by side read neighbouring heads of the same pages)
        part = at / per_group;
        if constexpr (LONE) sequence_position = shares.at[low];
        __syncthreads(); // (before the rings' first copies)
    }
    const bool whole = n_parts == 1;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u; // scores times a positive factor
    const float factor = a.scale == 0.0f ? 1.0f : fmaxf(fabsf(a.scale * 1.4426950408889634f), 1.17549435e-38f), slack = fminf(8.0f / factor, 1e30f);
    const int kvh = within % a.pool.kv_heads, block = within / a.pool.kv_heads;
    const int token0 = LONE ? unit : unit * a.tokens, tokens = LONE ? 1 : min(a.tokens, a.rows.n - token0), row0 = block * ROWS, rows = min(ROWS, tokens * mul - row0);
    const auto token_of = [&](int r) { return LONE ? 0 : (row0 + r) * a.of >> 16; };

    Segment only = {-1, 0, 0, 0, 0, 0}; // the first segment, which mostly is the only one
    if constexpr (LONE) { // every thread by itself
        int pos, s;
        if (a.ctas) {
            s = sequence_position.x;
            pos = sequence_position.y;
        } else {
            s = a.rows.place(token0, pos);
            pos = max(pos, -1);
        }
        if (s >= 0 && pos >= 0) {
            visible(pos, a.window, only.lo, only.hi);
            only.sequence = s;
            only.begin = only.lo / KT;
            only.end = (only.hi - 1) / KT + 1;
            only.tiles = only.end - only.begin;
        }
        if (tid == 0) { // (read behind the next barrier)
            seq_of[0] = s;
            pos_of[0] = pos;
            segment_of[0] = s >= 0 && pos >= 0 ? 0 : -1;
            segments[0] = only;
        }
    } else {
        if (tid < tokens) {
            int pos;
            const int s = a.rows.place(token0 + tid, pos);
            seq_of[tid] = s;
            pos_of[tid] = max(pos, -1);
        }
        __syncthreads();
        if (tid == 0) {
            int n = 0;
            segments_of_group(a, tokens, KT, [&](int t, int &pos) { pos = pos_of[t]; return seq_of[t]; }, [&](int i, int j, const Segment &sg) {
                for (int k = i; k < j; k++) segment_of[k] = sg.sequence < 0 ? -1 : n;
                if (sg.sequence >= 0) segments[n++] = sg;
            });
            n_segments = n;
        }
        __syncthreads();
        if (n_segments) only = segments[0];
    }

    const int total = LONE ? only.tiles : n_segments ? segments[n_segments - 1].tiles : 0;
    const int first = whole ? 0 : (int)((long long)total * part / n_parts), last = whole ? total : (int)((long long)total * (part + 1) / n_parts);

    const uint32_t ring = s32(smem) + warp * S * STAGE, q_at = s32(sQ);
    // this warp's tiles: numbers first + warp, + STEP_WARPS, .. of the list; `fetched` is the next to ask for
    int fetched = first + warp, seg_f = 0;
    Segment ahead = only;
    auto look_up = [&]() -> unsigned { // the number of the row that this lane looks up for the tile `fetched`
        if (fetched >= last) return NO_ROW;
        if constexpr (!LONE)
            while (ahead.tiles <= fetched) ahead = segments[++seg_f];
        const int pos = (ahead.end - (ahead.tiles - fetched)) * KT + lane;
        return lane < KT && pos >= ahead.lo && pos < ahead.hi ? row_at(a.pool, a.rows.table(ahead.sequence), pos, kvh) : NO_ROW;
    };
    unsigned row = look_up();
    auto fetch = [&](int stage) { // and look the next one up
        if (fetched < last) {
            const unsigned have = __ballot_sync(0xffffffffu, row != NO_ROW), row_0 = __shfl_sync(0xffffffffu, row, 0);
            if (lane == 0) there[warp][stage] = have;
            const uint32_t dst = ring + stage * STAGE;
            // rows one behind the other, as inside a page: one address, the others a fixed distance from it
            const bool together = 32 % PIECES == 0 && __all_sync(0xffffffffu, lane >= KT || (row != NO_ROW && row == row_0 + lane));
            if (together) {
                constexpr int RPI = 32 % PIECES == 0 ? 32 / PIECES : 1; // rows of a copy of the whole warp
                const int r0 = lane / PIECES, p = lane % PIECES;
                const size_t off = (size_t)(row_0 + r0) * RB + p * 16;
                const char *ks = (const char *)a.pool.keys + off, *vs = (const char *)a.pool.values + off;
                const uint32_t x = (uint32_t)(p ^ turn_of<HS>(r0)) << 4, to = dst + r0 * RB;
#pragma unroll
                for (int i = 0; i < KT / RPI; i++) {
                    const uint32_t at = to + RPI * i * RB + (x ^ turn_of<HS>(RPI * i) << 4); // (r0 and RPI i have no bit in common)
                    cp16(at, ks + RPI * i * RB);
                    cp16(at + KT * RB, vs + RPI * i * RB);
                }
            } else
#pragma unroll
                for (int i = 0; i < KT * PIECES / 32; i++) {
                    const int n = lane + 32 * i, r = n / PIECES, p = n % PIECES;
                    const unsigned from = __shfl_sync(0xffffffffu, row, r);
                    const size_t off = from == NO_ROW ? 0 : (size_t)from * RB + p * 16;
                    cp16_or_zeros(from != NO_ROW, dst + piece<HS>(r, p), (const char *)a.pool.keys + off);
                    cp16_or_zeros(from != NO_ROW, dst + KT * RB + piece<HS>(r, p), (const char *)a.pool.values + off);
                }
            fetched += STEP_WARPS;
            row = look_up();
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; i++) fetch(i);

    for (int i = tid; i < ROWS * PIECES; i += STEP_WARPS * 32) { // queries
        const int r = i / PIECES, c = i % PIECES, token = token_of(r);
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && a.scale != 0.0f && (LONE ? only.sequence : segment_of[token]) >= 0) { // (zeros for a row that sees nothing: padding may hold anything, and a NaN would reach the sums of the whole block)
            const uint16_t *q = (const uint16_t *)a.q + (long long)(token0 + token) * a.ldq + (size_t)(kvh * mul + row0 + r - token * mul) * HS + c * 8;
            if (a.vec) w = *reinterpret_cast<const uint4 *>(q);
            else w = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
        }
        *reinterpret_cast<uint4 *>(sQ + piece<HS>(r, c)) = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
    }
    __syncthreads();

    // rows 8 n + 2 t and 8 n + 2 t + 1 of this thread: what they see, within which segment
    int lo[NR][2], hi[NR][2], own[NR][2];
    int lo_most = only.lo, hi_least = only.hi;
    bool one = true; // every row of the block is of the first segment
    if constexpr (!LONE) {
        lo_most = 0;
        hi_least = INT_MAX;
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 8 * n + 2 * t + h, token = min(token_of(r), tokens - 1);
                lo[n][h] = hi[n][h] = 0;
                own[n][h] = r < rows ? segment_of[token] : 0;
                if (r < rows && own[n][h] >= 0) visible(pos_of[token], a.window, lo[n][h], hi[n][h]);
                if (r < rows && seq_of[token] >= 0) {
                    one &= own[n][h] == 0;
                    lo_most = max(lo_most, lo[n][h]);
                    hi_least = min(hi_least, hi[n][h]);
                }
            }
        one = __all_sync(0xffffffffu, one);
        lo_most = __reduce_max_sync(0xffffffffu, lo_most);
        hi_least = __reduce_min_sync(0xffffffffu, hi_least);
    }

    // ldmatrix rows: keys: lanes 0-15 rows 0-15 of a piece, 16-31 of the next; values (transposed): lanes 0-7 rows 0-7 of a piece, 8-15 of the next, 16-31 rows 8-15 likewise; queries:
    // lanes 0-7 rows 0-7 of a piece, 8-15, 16-23, 24-31 of the next three
    const int k_row = lane & 15, k_piece = lane >> 4, v_row = (lane & 7) + (lane >> 4 << 3), v_piece = lane >> 3 & 1, q_row = lane & 7, q_piece = lane >> 3;
    const uint32_t k_off = k_row * RB, k_x = (uint32_t)(k_piece ^ turn_of<HS>(k_row)) << 4, v_off = KT * RB + v_row * RB, v_x = (uint32_t)(v_piece ^ turn_of<HS>(v_row)) << 4;
    uint32_t qf[QREG ? NR : 1][QREG ? HS / 32 : 1][4]; // two steps of 16 entries each
    if constexpr (QREG)
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int k = 0; k < HS / 32; k++) ldmatrix4(q_at + piece<HS>(8 * n + q_row, 4 * k + q_piece), qf[n][k]);

    float o[NR][HS / 16][4], l[NR][2], top[NR][2], ref[NR][2]; // ref = top factor - LIFT
#pragma unroll
    for (int n = 0; n < NR; n++) {
#pragma unroll
        for (int i = 0; i < HS / 16; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        l[n][0] = l[n][1] = ref[n][0] = ref[n][1] = 0.0f;
        top[n][0] = top[n][1] = -CUDART_INF_F;
    }
    Segment sg = only;
    int seg = 0, stage = 0;
    bool huge = false; // a reference so large that it rounds by more than 2^-4 (the whole warp)
    for (int tile = first + warp; tile < last; tile += STEP_WARPS) {
        cp_wait<S - 2>();
        __syncwarp(); // and every lane has read the tile before, whose place the next copies take
        fetch(stage == 0 ? S - 1 : stage - 1);
        const uint32_t at = ring + stage * STAGE;
        float s[NR][KB][4];
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int b = 0; b < KB; b++) s[n][b][0] = s[n][b][1] = s[n][b][2] = s[n][b][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < HS / 32; k++) {
            uint32_t q[NR][4];
#pragma unroll
            for (int n = 0; n < NR; n++) {
                if constexpr (QREG) {
#pragma unroll
                    for (int i = 0; i < 4; i++) q[n][i] = qf[n][k][i];
                } else ldmatrix4(q_at + piece<HS>(8 * n + q_row, 4 * k + q_piece), q[n]);
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    uint32_t ka[4];
                    ldmatrix4(at + k_off + 16 * b * RB + (k_x ^ (2 * k + u) << 5), ka);
#pragma unroll
                    for (int n = 0; n < NR; n++) mma<T>(s[n][b], ka, q[n][2 * u], q[n][2 * u + 1]);
                }
        }
        const unsigned have = there[warp][stage];
        if constexpr (!LONE)
            while (sg.tiles <= tile) sg = segments[++seg];
        const int key0 = (sg.end - (sg.tiles - tile)) * KT;
        // masks; has the largest score of some row grown by too much?
        if (!(one && key0 >= lo_most && key0 + KT <= hi_least && have == (KT == 32 ? 0xffffffffu : (1u << (KT & 31)) - 1u)))
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int from = LONE ? lo_most - key0 : lo[n][h] - key0, to = LONE ? hi_least - key0 : own[n][h] == seg ? hi[n][h] - key0 : INT_MIN;
#pragma unroll
                    for (int b = 0; b < KB; b++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int j = 16 * b + 8 * i + g;
                            if (!(j >= from && j < to && (have >> j & 1u))) s[n][b][2 * i + h] = -CUDART_INF_F;
                        }
                }
        const auto highest = [&](int n, int h) {
            float mx = s[n][0][h];
#pragma unroll
            for (int b = 0; b < KB; b++) mx = fmaxf(mx, fmaxf(s[n][b][h], s[n][b][2 + h]));
            return mx;
        };
        bool higher = false;
#pragma unroll
        for (int n = 0; n < NR; n++) higher |= highest(n, 0) > top[n][0] + slack || highest(n, 1) > top[n][1] + slack;
        if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float mx = highest(n, h);
#pragma unroll
                    for (int i = 4; i < 32; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
                    if (mx > top[n][h]) {
                        const float next = mx * factor - LIFT, f = top[n][h] == -CUDART_INF_F ? 0.0f : ex2(ref[n][h] - next);
                        top[n][h] = mx;
                        ref[n][h] = next;
                        l[n][h] *= f;
#pragma unroll
                        for (int i = 0; i < HS / 16; i++) { o[n][i][h] *= f; o[n][i][2 + h] *= f; }
                    }
                    huge |= fabsf(ref[n][h]) > 1048576.0f;
                }
            huge = __any_sync(0xffffffffu, huge);
        }
        // An exponent is the scaled score, not yet rounded, minus a reference that is: where that rounds by hundreds every probability of the row would be 0, or infinite.  There scores are rounded like it first.
        if (huge)
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[n][b][i] *= factor;
        const float by = huge ? 1.0f : factor;
        uint32_t pp[PARTS][NR][KB][2]; // of 8 positions each: of positions 2 t, 2 t + 1 and row g
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float p0 = ex2(fmaf(s[n][b][2 * i], by, -ref[n][0])), p1 = ex2(fmaf(s[n][b][2 * i + 1], by, -ref[n][1]));
                    l[n][0] += p0;
                    l[n][1] += p1;
                    float2 left = make_float2(p0, p1);
#pragma unroll
                    for (int c = 0; c < PARTS; c++) {
                        const uint32_t w = pack2<T>(left.x, left.y);
                        pp[c][n][b][i] = transpose8x8(w);
                        const float2 r = unpack2<T>(w);
                        left = make_float2(left.x - r.x, left.y - r.y);
                    }
                }
#pragma unroll
        for (int i = 0; i < HS / 16; i++) {
            // The products cut what they add to their sums.  With FP32 results a tile's are made from zero and added as FP32 numbers are, so that a long row's sums do not drift.
            float tile_o[NR][4];
            if constexpr (PARTS > 1)
#pragma unroll
                for (int n = 0; n < NR; n++) tile_o[n][0] = tile_o[n][1] = tile_o[n][2] = tile_o[n][3] = 0.0f;
#pragma unroll
            for (int b = 0; b < KB; b++) {
                uint32_t va[4];
                ldmatrix4_trans(at + v_off + 16 * b * RB + (v_x ^ i << 5), va);
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int c = 0; c < PARTS; c++) mma<T>(PARTS > 1 ? tile_o[n] : o[n][i], va, pp[c][n][b][0], pp[c][n][b][1]);
            }
            if constexpr (PARTS > 1)
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int u = 0; u < 4; u++) o[n][i][u] += tile_o[n][u];
        }
        if (++stage == S) stage = 0;
    }
    cp_wait<0>();

    // ---- join: warps, then (through the workspace) CTAs ----
    __syncthreads(); // the rings are free
    float *parts = reinterpret_cast<float *>(smem);
    float sum = 0.0f; // not finite where an entry is not
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float all = l[n][h];
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) all += __shfl_xor_sync(0xffffffffu, all, i);
            const int r = 8 * n + 2 * t + h;
            if (g == 0) { wref[warp][r] = top[n][h] == -CUDART_INF_F ? -CUDART_INF_F : ref[n][h]; wsum[warp][r] = all; }
            if (r < rows) {
                float *to = parts + (warp * ROWS + r) * part_stride(HS) + g;
#pragma unroll
                for (int i = 0; i < HS / 16; i++) {
                    to[16 * i] = o[n][i][h];
                    to[16 * i + 8] = o[n][i][2 + h];
                    sum += 0.0f * o[n][i][h] + 0.0f * o[n][i][2 + h];
                }
            }
        }
    __syncwarp();
    if (__any_sync(0xffffffffu, sum != 0.0f))
        slow_rows<HS, T>(a, sQ, rows, row0, token0, kvh, first, last, warp, segments, segment_of, pos_of, factor, parts + warp * ROWS * part_stride(HS), wref[warp], wsum[warp]);
    __syncthreads();
    if (tid < rows) {
        const int token = token_of(tid), head = kvh * mul + row0 + tid - token * mul;
        float M = -CUDART_INF_F, L = 0.0f;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) M = fmaxf(M, wref[w][tid]);
        const float base = M == -CUDART_INF_F ? 0.0f : M;
        float f[STEP_WARPS];
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) {
            f[w] = wref[w][tid] == M ? 1.0f : ex2(wref[w][tid] - base);
            L = fmaf(f[w], wsum[w][tid], L);
        }
        if (!whole) stats_of<HS, NR>(a, groups)[(size_t)blockIdx.x * ROWS + tid] = make_float2(M, L);
        const float scale = whole ? 1.0f / L : 1.0f;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) weight[w][tid] = L == 0.0f ? 0.0f : f[w] * scale; // nothing seen: zeros
    }
    __syncthreads();
    for (int i = tid; i < rows * (HS / 4); i += STEP_WARPS * 32) {
        const int r = i / (HS / 4), e = i % (HS / 4) * 4, token = token_of(r);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) {
            const float f = weight[w][r];
            const float4 p = *reinterpret_cast<const float4 *>(parts + (w * ROWS + r) * part_stride(HS) + e);
            x = make_float4(fmaf(f, p.x, x.x), fmaf(f, p.y, x.y), fmaf(f, p.z, x.z), fmaf(f, p.w, x.w));
        }
        if (!whole) *reinterpret_cast<float4 *>(a.work + ((size_t)blockIdx.x * ROWS + r) * HS + e) = x;
        else if (seq_of[token] >= 0) put_results(a, token0 + token, kvh * mul + row0 + r - token * mul, HS, e, x);
    }
}

// Joins the parts of units that several CTAs shared, and clears rows that see nothing.  FEW (where a unit has few CTAs): eight rows a CTA, four entries a thread, part by part; else a row a
// CTA, whose HS / 4 threads a part take parts in turn.
template <int HS, int NR, bool LONE, bool FEW> __global__ void __launch_bounds__(128) k_paged_join_shares(const Step a) {
    constexpr int ROWS = step_rows(NR), LANES = HS / 4, GROUPS = 128 / LANES, AT_ONCE = 128;
    pdl_wait();
    const int tid = threadIdx.x, per_group = a.pool.kv_heads * a.blocks, group = blockIdx.x / per_group, within = blockIdx.x % per_group, groups = (a.rows.n + a.tokens - 1) / a.tokens;
    const int kvh = within % a.pool.kv_heads, block = within / a.pool.kv_heads, token0 = group * a.tokens, tokens = min(a.tokens, a.rows.n - token0), row0 = block * ROWS, rows = min(ROWS, tokens * a.mul - row0);
    const int *plan = plan_of<HS, NR>(a, groups);
    const int before = plan[group], parts = (plan[group + 1] - before) / per_group;
    if (parts == 1) return; // one CTA's
    const auto place = [&](int r, int &row, int &head) {
        const int token = LONE ? 0 : (row0 + r) / a.mul;
        row = token0 + token;
        head = kvh * a.mul + row0 + r - token * a.mul;
        int pos;
        return a.rows.place(row, pos) >= 0;
    };
    const auto slot = [&](int p) { return (size_t)(before + p * per_group + within) * ROWS; };
    const float2 *stats = stats_of<HS, NR>(a, groups);
    int row, head;
    if constexpr (FEW) {
        for (int i = tid; i < 8 * LANES; i += 128) {
            const int r = blockIdx.y * 8 + i / LANES, e = i % LANES * 4;
            if (r >= rows || !place(r, row, head)) continue;
            float M = -CUDART_INF_F, L = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int p = 0; p < parts; p++) {
                const float2 st = stats[slot(p) + r];
                const float4 v = *reinterpret_cast<const float4 *>(a.work + (slot(p) + r) * HS + e);
                const float grown = fmaxf(M, st.x), base = grown == -CUDART_INF_F ? 0.0f : grown, f = M == grown ? 1.0f : ex2(M - base), w = st.x == grown ? 1.0f : ex2(st.x - base);
                M = grown;
                L = fmaf(w, st.y, L * f);
                x = make_float4(fmaf(w, v.x, x.x * f), fmaf(w, v.y, x.y * f), fmaf(w, v.z, x.z * f), fmaf(w, v.w, x.w * f));
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            put_results(a, row, head, HS, e, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        }
    } else {
        __shared__ float2 stat[AT_ONCE];
        __shared__ float red[4], sums_l[GROUPS];
        __shared__ float4 sums[GROUPS][LANES];
        const int r = blockIdx.y, lane = tid % LANES, mine = tid / LANES;
        if (r >= rows || !place(r, row, head)) return;
        float M = -CUDART_INF_F, L = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p0 = 0; p0 < parts; p0 += AT_ONCE) { // (more than 128 parts: what was joined so far is moved to the larger reference)
            const int n = min(AT_ONCE, parts - p0);
            const float2 st = tid < n ? stats[slot(p0 + tid) + r] : make_float2(-CUDART_INF_F, 0.0f);
            const float most = warp_max_f(st.x);
            __syncthreads();
            if (tid % 32 == 0) red[tid / 32] = most;
            __syncthreads();
            const float grown = fmaxf(M, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), base = grown == -CUDART_INF_F ? 0.0f : grown, f = M == grown ? 1.0f : ex2(M - base);
            M = grown;
            L *= f;
            x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
            stat[tid] = make_float2(st.x == M ? 1.0f : ex2(st.x - base), st.y);
            __syncthreads();
            if (mine < GROUPS)
#pragma unroll 8
                for (int p = mine; p < n; p += GROUPS) {
                    const float4 v = *reinterpret_cast<const float4 *>(a.work + (slot(p0 + p) + r) * HS + lane * 4);
                    const float2 w = stat[p];
                    L = fmaf(w.x, w.y, L);
                    x = make_float4(fmaf(w.x, v.x, x.x), fmaf(w.x, v.y, x.y), fmaf(w.x, v.z, x.z), fmaf(w.x, v.w, x.w));
                }
        }
        if (mine < GROUPS) {
            sums[mine][lane] = x;
            if (lane == 0) sums_l[mine] = L;
        }
        __syncthreads();
        if (tid < LANES) {
#pragma unroll
            for (int i = 1; i < GROUPS; i++) {
                const float4 p = sums[i][lane];
                x = make_float4(x.x + p.x, x.y + p.y, x.z + p.z, x.w + p.w);
                L += sums_l[i];
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            put_results(a, row, head, HS, lane * 4, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        }
    }
}

// Joins the parts of a row's head, at most 32 of them: a warp each, the weight of a part a lane.
template <int HS> __global__ void __launch_bounds__(128) k_paged_join_few(const Step a) {
    constexpr int V = HS % 128 == 0 ? 4 : HS % 64 == 0 ? 2 : 1, N = HS / (32 * V); // entries of a lane at a time, how many times
    pdl_wait();
    const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5), row = item / a.heads, head = item % a.heads;
    int pos;
    if (row >= a.rows.n || a.rows.place(row, pos) < 0) return;
    const float *part = a.work + (size_t)item * a.splits * HS;
    const float2 st = lane < a.splits ? (reinterpret_cast<const float2 *>(a.work + (size_t)a.rows.n * a.heads * a.splits * HS) + (size_t)item * a.splits)[lane] : make_float2(-CUDART_INF_F, 0.0f);
    const float M = warp_max_f(st.x), base = M == -CUDART_INF_F ? 0.0f : M, f = st.x == M ? 1.0f : ex2(st.x - base);
    const unsigned some = __ballot_sync(0xffffffffu, st.y != 0.0f); // (what the entries of a part without a sum hold is not defined)
    float L = st.y != 0.0f ? f * st.y : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    float x[N][V];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < V; i++) x[n][i] = 0.0f;
    for (int s = 0; s < a.splits; s++) {
        const float w = __shfl_sync(0xffffffffu, f, s);
        if (!(some >> s & 1u)) continue;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float *p = part + (size_t)s * HS + (n * 32 + lane) * V;
            float v[V];
            if constexpr (V == 4) { const float4 u = *reinterpret_cast<const float4 *>(p); v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w; }
            else if constexpr (V == 2) { const float2 u = *reinterpret_cast<const float2 *>(p); v[0] = u.x; v[1] = u.y; }
            else v[0] = *p;
#pragma unroll
            for (int i = 0; i < V; i++) x[n][i] = fmaf(w, v[i], x[n][i]);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int n = 0; n < N; n++) {
        const long long at = row * a.ldo + (long long)head * HS + (n * 32 + lane) * V;
#pragma unroll
        for (int i = 0; i < V; i++) x[n][i] *= inv;
        if constexpr (V == 4) put_results(a, row, head, HS, (n * 32 + lane) * 4, make_float4(x[n][0], x[n][1], x[n][2], x[n][3]));
        else
#pragma unroll
            for (int i = 0; i < V; i++) {
                if (a.out_type == B200_GGML_F32) ((float *)a.out)[at + i] = x[n][i];
                else if (a.out_type == B200_GGML_F16) put((__half *)a.out + at + i, x[n][i]);
                else put((bf16 *)a.out + at + i, x[n][i]);
            }
    }
}

// Joins the parts of a row's head: 128 threads, 4 entries each, HS / 4 threads a part.  At most MAX_SPLITS parts.
constexpr int MAX_SPLITS = 296;
template <int HS> __global__ void __launch_bounds__(128) k_paged_join(const Step a) {
    constexpr int LANES = HS / 4, GROUPS = 128 / LANES;
    __shared__ float weight[MAX_SPLITS], red[2][4];
    __shared__ float4 sums[GROUPS][LANES];
    pdl_wait();
    const int tid = threadIdx.x, row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    int pos;
    if (a.rows.place(row, pos) < 0) return;
    const size_t at = ((size_t)row * a.heads + head) * a.splits;
    const float2 *stat = reinterpret_cast<const float2 *>(a.work + (size_t)a.rows.n * a.heads * a.splits * HS) + at;
    const float4 *part = reinterpret_cast<const float4 *>(a.work + at * HS);
    float2 st[(MAX_SPLITS + 127) / 128];
    float M = -CUDART_INF_F, L = 0.0f;
#pragma unroll
    for (int i = 0; i < (MAX_SPLITS + 127) / 128; i++) {
        st[i] = tid + 128 * i < a.splits ? stat[tid + 128 * i] : make_float2(-CUDART_INF_F, 0.0f);
        M = fmaxf(M, st[i].x);
    }
    M = warp_max_f(M);
    if (tid % 32 == 0) red[0][tid / 32] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float base = M == -CUDART_INF_F ? 0.0f : M;
#pragma unroll
    for (int i = 0; i < (MAX_SPLITS + 127) / 128; i++) {
        const bool some = st[i].y != 0.0f; // (what the entries of a part without a sum hold is not defined)
        const float f = st[i].x == M ? 1.0f : ex2(st[i].x - base);
        if (tid + 128 * i < a.splits) weight[tid + 128 * i] = some ? f : -1.0f;
        L += some ? f * st[i].y : 0.0f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (tid % 32 == 0) red[1][tid / 32] = L;
    __syncthreads();
    L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const int lane = tid % LANES, group = tid / LANES;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (group < GROUPS)
        for (int s = group; s < a.splits; s += GROUPS) {
            const float f = weight[s];
            if (f < 0.0f) continue;
            const float4 p = part[(size_t)s * LANES + lane];
            x = make_float4(fmaf(f, p.x, x.x), fmaf(f, p.y, x.y), fmaf(f, p.z, x.z), fmaf(f, p.w, x.w));
        }
    if (group < GROUPS) sums[group][lane] = x;
    __syncthreads();
    if (tid < LANES) {
#pragma unroll
        for (int i = 1; i < GROUPS; i++) {
            const float4 p = sums[i][lane];
            x = make_float4(x.x + p.x, x.y + p.y, x.z + p.z, x.w + p.w);
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        put_results(a, row, head, HS, lane * 4, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    }
}

} // namespace paged
