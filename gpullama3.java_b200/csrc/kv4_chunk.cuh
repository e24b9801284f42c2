// kv4_chunk.cuh -- attention of prompt chunks over the 4-bit cache on the 5th-generation tensor cores, with 16-bit results.
//
// A CTA takes 128 rows (tokens x query heads of one key/value head) and runs through the positions that any of them sees, 128 at a time:
//   warps 16-23  turn a tile's records (one a warp) into FP16 operands in shared memory: keys [position][entry], values transposed [entry][position], both K-major
//   warp 24      issues S = Q K^T and O += P V, with P read from TMEM
//   warps 0-15   exponentials, two threads a row; P as FP16 takes the place of S; O is scaled where a row's maximum has grown by too much, which is rare
// A tile's work is a chain: scores, exponentials, product, about 5000 cycles of which 1024 are the tensor cores' and 1024 the exponentials' (16 a cycle).  So even and odd tiles are two
// streams with accumulators, maxima and sums of their own, each of eight warps, which the end joins: while one waits for its products the other computes.  Heads of 128, two streams of
// scores and results: all 512 columns of TMEM.
// Measured (512 tokens, 32 heads over 8 of 128, 8192 positions: 66.6 GFLOP): 104 us (99-109 from box to box), 640 TFLOP/s, 38 % of the 1690 measured.  A tile takes 2300 cycles: its 16
// products 1400 (1024 were nothing else at shared memory), beside them the conversion of its records, one a warp, 2400 with what it waits for; 0.57 instructions a cycle and scheduler.
// One stream with two S and a maximum agreed on by a row's threads in every tile took 116-123 us; 256 rows a CTA with half the conversions 133 us (two blocks of rows in place of the two
// streams; 64 pairs of CTAs whose parts had to be joined).
// Rounding: queries (times a power of two), keys, values and probabilities are FP16 operands, sums are FP32.  Entries of a position outside FP16 (a scale above 8184: codes of up to 8 times
// that) become operands times 2^-5, and the position's scores, or its probabilities as operands, times 2^5.  A value's NaN stays out of the product, where 0 * NaN would reach every row: the
// rows that see it note its group, and write NaN there.  The append marks the slots that have taken such an entry (kv4.cuh), and only CTAs that meet a marked slot look for them: looked for in
// every tile they cost 9 % (104 us became 113); so the time of other slots is what it was, and 123 us in place of 97 for calls back to back where one position of a marked slot is such a one.
//
// Rows of a tile may belong to several slots and stand in any order: a run of tokens of one slot is a segment, the tiles of all segments are one list, and a row masks what is not its own.
// Every wait is bounded: after two seconds the CTA gives up, waits for its products under way, frees its tensor memory and, whichever warp it was, writes the cache's error word.
#pragma once
#include <type_traits>

#include "kv4.cuh"

namespace kv4 {

constexpr int CHUNK_ROWS = 128, CHUNK_KEYS = 128, CHUNK_K_STAGES = 3, CHUNK_V_STAGES = 2, CHUNK_RECORDS = CHUNK_KEYS / BLOCK;
constexpr int CHUNK_SOFTMAX = 16, CHUNK_DEQUANT = CHUNK_RECORDS, CHUNK_ISSUER = CHUNK_SOFTMAX + CHUNK_DEQUANT, CHUNK_THREADS = (CHUNK_ISSUER + 1) * 32; // warps of each kind
__host__ __device__ constexpr int chunk_tile_bytes(int hs) { return hs * CHUNK_KEYS * 2; } // of queries, keys or values

struct Segment { // a run of tokens of one slot and the records that any of them sees
    int slot, begin, end, tiles; // records [begin, end); tiles of all segments up to and with this one
};
struct ChunkSmem { // behind the operands
    uint4 odd[CHUNK_K_STAGES][CHUNK_RECORDS]; // by record of the keys' stage: x: positions whose keys (low half) or values (high half) are held times 2^-5; y, z: whose values are NaN, 16 bits a group; w: any
    unsigned long long k_full[CHUNK_K_STAGES], k_free[CHUNK_K_STAGES], v_full[CHUNK_V_STAGES], v_free[CHUNK_V_STAGES];
    unsigned long long s_full[2], p_full[2], drained; // by stream
    unsigned long long pair[CHUNK_SOFTMAX / 2];       // the two warps that share a stream's rows
    unsigned tmem, bail, again[2], repeat[2], marked; // again: a row's maximum has to move; repeat: these are the scores of the tile before once more; marked: a token's slot is
    int n_segments, single;
    int slot[CHUNK_ROWS], pos[CHUNK_ROWS], segment[CHUNK_ROWS]; // by token
    unsigned nan[CHUNK_ROWS];                                   // by row: groups in which it has seen a NaN
    float factor[CHUNK_ROWS];                                   // by row: what turns a product into a score in units of log2
    float half_row[2][2][CHUNK_ROWS];                           // by stream: what the two threads of a row tell each other, their sums at the end
    float top[2][CHUNK_ROWS];
    Segment segments[CHUNK_ROWS];
};
__host__ __device__ constexpr size_t chunk_smem_bytes(int hs) { return 1024 + (1 + CHUNK_K_STAGES + CHUNK_V_STAGES) * chunk_tile_bytes(hs) + sizeof(ChunkSmem); }

__device__ __forceinline__ uint32_t s32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(const void *bar, unsigned n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(bar)), "r"(n)); }
__device__ __forceinline__ void bar_arrive(const void *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(bar)) : "memory"); }
constexpr unsigned WAIT_TRIES = 1u << 19; // about two seconds of a warp's own time: a try sleeps for some 4 us where nothing comes (2^25 of them took minutes)
__device__ __forceinline__ bool bar_passed(uint32_t bar, unsigned parity) {
    unsigned done;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0u;
}
// false: given up.  Warps that may come late sleep between tries: a dozen of them asking all the time took the issue slots of the one that issues the products.
template <bool SLEEP = true> __device__ __forceinline__ bool bar_wait(const void *bar, unsigned parity, volatile unsigned *bail) {
    const uint32_t b = s32(bar);
    for (unsigned i = 1; i < WAIT_TRIES; i++) {
        if (bar_passed(b, parity)) return true;
        if (SLEEP) __nanosleep(20);
        if ((i & 1023u) == 0u && *bail) return false;
    }
    *bail = 1u;
    return false;
}
// K-major operand descriptors: start >> 4 | 1 << 16 | 8 rows >> 4 << 32 | version 1 << 46 | swizzle (2: rows of 128 bytes, 4: rows of 64) << 61
__device__ __forceinline__ uint64_t desc128(uint32_t a) { return (uint64_t)((a & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61); }
__device__ __forceinline__ uint64_t desc64(uint32_t a) { return (uint64_t)((a & 0x3ffffu) >> 4) | (1ull << 16) | (32ull << 32) | (1ull << 46) | (4ull << 61); }
// The warp that issues products runs as one, so that addresses stay in its uniform registers, and one lane (lead) does it: with a single thread in that branch every operand went through
// vector registers, and the eight products of a step took twice their time to issue.
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t lead) {
    asm volatile("{.reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t lead) { // the first operand from TMEM
    asm volatile("{.reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(const void *bar, uint32_t lead) {
    asm volatile("{.reg .pred q; setp.ne.b32 q, %1, 0; @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];}" ::"r"(s32(bar)), "r"(lead) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t a, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(a));
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Two FP32 operations in one.
__device__ __forceinline__ unsigned long long pack_f32x2(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(unsigned long long v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void store_matrices(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) { // four of 8 x 8 halves; lane l gives the address of row l % 8 of matrix l / 8
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// What a dequantising lane holds of a record: codes of both halves, the key scales of positions g and g + 8, the value scales of positions 2 t, 2 t + 8 and 2 t + 1, 2 t + 9.
template <int HS> struct Raw {
    static constexpr int NG = groups(HS), VW = vec_words(HS);
    uint32_t k[2][NG], v[2][NG], ks[NG], vs[2][NG];
    __device__ __forceinline__ void load(const unsigned char *rec, int lane) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(rec), *s = w + 4 * HS;
        const int g = lane >> 2, t = lane & 3;
        uint32_t x[VW];
        auto get = [&](const uint32_t *p, uint32_t *to) {
            lds_words<VW>(p, x);
#pragma unroll
            for (int i = 0; i < VW; i++) to[i] = x[i];
        };
#pragma unroll
        for (int c = 0; c < NG / VW; c++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                get(w + word_of<HS>(half, lane, c * VW), k[half] + c * VW);
                get(w + 2 * HS + word_of<HS>(half, lane, c * VW), v[half] + c * VW);
            }
            get(s + g * NG + c * VW, ks + c * VW);
            get(s + 8 * NG + 2 * t * NG + c * VW, vs[0] + c * VW);
            get(s + 8 * NG + (2 * t + 1) * NG + c * VW, vs[1] + c * VW);
        }
    }
};

struct Chunk {
    Step step;
    int tokens;      // of a CTA: 128 / (query heads of a key/value head)
    int splits;      // CTAs that share a tile of rows
    int vec_out;     // result rows start on 16-byte boundaries
    unsigned *error; // the cache's error word (mapped host memory)
};

// GIVE_UP (tests): for their last wait, that for the products that end a stream, the warps of the rows wait for a barrier at which nobody arrives.
template <int HS, bool GIVE_UP = false> __global__ void __launch_bounds__(CHUNK_THREADS, 1) k_chunk(const Chunk c) {
    constexpr int NG = groups(HS);
    extern __shared__ unsigned char raw_smem[];
    unsigned char *smem = raw_smem + (-s32(raw_smem) & 1023u); // the operands' swizzle counts from 1024-byte boundaries
    unsigned char *sQ = smem, *sK = sQ + chunk_tile_bytes(HS), *sV = sK + CHUNK_K_STAGES * chunk_tile_bytes(HS);
    ChunkSmem &sh = *reinterpret_cast<ChunkSmem *>(sV + CHUNK_V_STAGES * chunk_tile_bytes(HS));
    const Step &a = c.step;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int G = a.kv.kv_heads, mul = a.heads / G;
    const unsigned of = (65535u + mul) / mul; // r / mul = r of >> 16: exact, as r mul < 2^16
    const auto token_of = [&](int r) { return (int)(r * of >> 16); };
    const int n_tiles = (a.rows.n + c.tokens - 1) / c.tokens;
    const int split = blockIdx.x % c.splits, kvh = blockIdx.x / c.splits % G, tile = n_tiles - 1 - blockIdx.x / c.splits / G; // the last tokens, which see most, first
    const int token0 = tile * c.tokens, tokens = min(c.tokens, a.rows.n - token0);

    pdl_wait();
    if (tid == 0) {
        for (int i = 0; i < CHUNK_K_STAGES; i++) {
            bar_init(&sh.k_full[i], CHUNK_DEQUANT);
            bar_init(&sh.k_free[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            bar_init(&sh.v_full[i], CHUNK_DEQUANT);
            bar_init(&sh.v_free[i], 1);
            bar_init(&sh.s_full[i], 1);
            bar_init(&sh.p_full[i], CHUNK_SOFTMAX / 2);
            sh.again[i] = sh.repeat[i] = 0;
        }
        for (int i = 0; i < CHUNK_SOFTMAX / 2; i++) bar_init(&sh.pair[i], 2);
        bar_init(&sh.drained, 1);
        sh.bail = sh.marked = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == CHUNK_SOFTMAX) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid < CHUNK_ROWS) {
        int slot = -1, pos = -1;
        if (tid < tokens) {
            slot = a.rows.slot_of(token0 + tid);
            pos = a.rows.position(token0 + tid);
            if (slot < 0 || slot >= a.kv.slots || pos >= a.kv.context) slot = pos = -1; // padding
            pos = max(pos, -1); // (positions are subtracted from, and both warps of a row have to find the same)
        }
        sh.slot[tid] = slot;
        sh.pos[tid] = pos;
        sh.segment[tid] = -1;
        sh.nan[tid] = 0;
    }
    // queries: a row a warp, all of a warp's rows under way at once
    constexpr int WARPS = CHUNK_THREADS / 32, QROWS = (CHUNK_ROWS + WARPS - 1) / WARPS;
    float4 x[QROWS]; // entries 4 lane .. + 3
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const int r = warp + i * WARPS, token = token_of(r);
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (token < tokens && r < CHUNK_ROWS && lane * 4 < HS) {
            const float *q = a.q + (long long)(token0 + token) * a.ldq + (size_t)(kvh * mul + r - token * mul) * HS + lane * 4;
            if (a.vec) x[i] = *reinterpret_cast<const float4 *>(q);
            else x[i] = make_float4(q[0], q[1], q[2], q[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const int r = warp + i * WARPS;
        if (r >= CHUNK_ROWS) break;
        const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w)))))); // (not below 0: its bits are in order)
        const int e = min(max((int)(__float_as_uint(top) >> 23), 12), 230); // times a power of two: below 1024, whatever its size; with the sign of the scale
        const float up = a.scale == 0.0f ? 0.0f : copysignf(__uint_as_float((unsigned)(263 - e) << 23), a.scale), down = __uint_as_float((unsigned)(e - 9) << 23);
        if (lane * 4 < HS)
            *reinterpret_cast<uint2 *>(sQ + (lane / 8) * (CHUNK_ROWS * 64) + r * 64 + (((lane % 8 / 2) ^ (r >> 1 & 3)) << 4) + (lane & 1) * 8) =
                make_uint2(pack_f16(x[i].x * up, x[i].y * up), pack_f16(x[i].z * up, x[i].w * up));
        if (lane == 0) sh.factor[r] = a.scale == 0.0f ? 1.0f : fmaxf(down * fabsf(a.scale * 1.4426950408889634f), 1.17549435e-38f); // (0 times -inf is a NaN)
    }
    __syncthreads();
    if (tid < tokens && sh.slot[tid] >= 0 && a.kv.odd[sh.slot[tid]] != 0u) sh.marked = 1u;
    if (tid == CHUNK_ROWS && a.kv.odd[a.kv.slots] != 0u) sh.bail = 1u; // an earlier CTA has given up: none waits as long again
    if (warp == 0) { // one slot for all, as inside a prompt: one segment
        bool same = sh.slot[0] >= 0;
        int from = INT32_MAX, to = 0;
        for (int i = lane; i < tokens; i += 32) {
            int lo, hi;
            visible(sh.pos[i], a.window, lo, hi);
            same &= sh.slot[i] == sh.slot[0];
            if (hi > lo) { from = min(from, lo); to = max(to, hi); }
        }
        same = __all_sync(0xffffffffu, same);
        from = __reduce_min_sync(0xffffffffu, from);
        to = __reduce_max_sync(0xffffffffu, to);
        if (same && to > 0) {
            for (int i = lane; i < tokens; i += 32) sh.segment[i] = 0;
            if (lane == 0) {
                const int begin = from / BLOCK, end = (to + BLOCK - 1) / BLOCK;
                sh.segments[0] = {sh.slot[0], begin, end, (end - begin + CHUNK_RECORDS - 1) / CHUNK_RECORDS};
                sh.n_segments = 1;
            }
        }
        if (lane == 0) sh.single = same && to > 0;
    }
    if (tid == 0 && !sh.single) {
        int n = 0, total = 0;
        for (int i = 0; i < tokens;) {
            const int slot = sh.slot[i];
            int j = i, from = INT32_MAX, to = 0;
            for (; j < tokens && sh.slot[j] == slot; j++) {
                int lo, hi;
                visible(sh.pos[j], a.window, lo, hi);
                if (hi > lo) { from = min(from, lo); to = max(to, hi); }
                sh.segment[j] = n;
            }
            if (slot >= 0 && to > 0) {
                const int begin = from / BLOCK, end = (to + BLOCK - 1) / BLOCK;
                total += (end - begin + CHUNK_RECORDS - 1) / CHUNK_RECORDS;
                sh.segments[n++] = {slot, begin, end, total};
            } else
                for (int k = i; k < j; k++) sh.segment[k] = -1;
            i = j;
        }
        sh.n_segments = n;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the queries, for the products
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0), tS = tmem, tO = tmem + 2 * CHUNK_KEYS;
    const int total = __shfl_sync(0xffffffffu, sh.n_segments ? sh.segments[sh.n_segments - 1].tiles : 0, 0);
    const int first = (int)((long long)total * split / c.splits), last = (int)((long long)total * (split + 1) / c.splits), count = last - first;

    if (warp >= CHUNK_SOFTMAX && warp < CHUNK_ISSUER) {
        // ===== records -> FP16 operands =====
        const int w = warp - CHUNK_SOFTMAX, g = lane >> 2, t = lane & 3;
        const uint32_t one = magic();
        int seg = 0, ahead = 0, block = 0, stop = 0, behind = 0; // tiles left in the segment, this warp's record in the next one, the segment's end; raw is a record behind it
        if (count > 0) {
            while (sh.segments[seg].tiles <= first) seg++;
            const int before = seg ? sh.segments[seg - 1].tiles : 0;
            ahead = sh.segments[seg].tiles - first;
            block = sh.segments[seg].begin + (first - before) * CHUNK_RECORDS + w;
            stop = sh.segments[seg].end;
        }
        Raw<HS> raw;
        auto fetch = [&] { // this warp's record of the list's next tile; behind the segment's end its last one, whose values then count as zeros
            if (ahead == 0) {
                seg++;
                ahead = sh.segments[seg].tiles - sh.segments[seg - 1].tiles;
                block = sh.segments[seg].begin + w;
                stop = sh.segments[seg].end;
            }
            behind = block >= stop;
            const unsigned char *rec = record<HS>(a.kv, sh.segments[seg].slot, kvh, min(block, stop - 1));
            raw.load(rec, lane);
            ahead--;
            block += CHUNK_RECORDS;
            if (block < stop && lane < (record_bytes(HS) + 127) / 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(rec + (size_t)CHUNK_RECORDS * record_bytes(HS) + min(lane * 128, record_bytes(HS) - 1)));
        };
        // rows 16 w + 8 half + g of the keys; positions 16 w + 8 half + 2 t, + 1 of the values: 16-byte chunk 2 (w % 4) + half of the rows of 64 positions
        const uint32_t k_at = s32(sK) + (w * 16 + g) * 64 + ((t ^ (g >> 1 & 3)) << 4);
        const uint32_t v_at = s32(sV) + (w / 4) * (HS * 128) + lane * 128 + ((w % 4 * 2 ^ (lane & 7)) << 4);
        if (count > 0) fetch();
        int ks = 0; // stage of the keys
        unsigned k_phase = 1;
        for (int j = 0; j < count; j++) {
            const int b = j & 1;
            uint32_t v[2][NG], dv[2][NG]; // the values' codes and scales
#pragma unroll
            for (int i = 0; i < NG; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    v[h][i] = raw.v[h][i];
                    dv[h][i] = __byte_perm(raw.vs[0][i], raw.vs[1][i], h ? 0x7632 : 0x5410);
                }
            if (behind)
#pragma unroll
                for (int i = 0; i < NG; i++) dv[0][i] = dv[1][i] = 0u;
            if (j >= CHUNK_K_STAGES && !__all_sync(0xffffffffu, bar_wait(&sh.k_free[ks], k_phase, &sh.bail))) break; // the scores of tile j - 3 stand
            if (__any_sync(0xffffffffu, sh.marked != 0u)) { // entries that FP16 does not hold, and NaN
                const auto wide = [](uint32_t d) { return d > KV4_ODD && d <= 0x7c00u; };
                uint32_t w5 = 0, nan[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    w5 |= (wide(raw.ks[i] & 0x7fffu) ? 1u << g : 0u) | (wide(raw.ks[i] >> 16 & 0x7fffu) ? 0x100u << g : 0u);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t a0 = dv[h][i] & 0x7fffu, a1 = dv[h][i] >> 16 & 0x7fffu, at = 8 * h + 2 * t;
                        w5 |= (wide(a0) ? 0x10000u << at : 0u) | (wide(a1) ? 0x20000u << at : 0u);
                        nan[i / 2] |= ((a0 > 0x7c00u ? 1u << at : 0u) | (a1 > 0x7c00u ? 2u << at : 0u)) << (16 * (i & 1));
                        dv[h][i] &= (a0 > 0x7c00u ? 0u : 0xffffu) | (a1 > 0x7c00u ? 0u : 0xffff0000u);
                    }
                }
                w5 = __reduce_or_sync(0xffffffffu, w5);
                nan[0] = __reduce_or_sync(0xffffffffu, nan[0]);
                nan[1] = __reduce_or_sync(0xffffffffu, nan[1]);
                const auto scale = [&](int lo, int hi) { return (w5 >> lo & 1u ? 0x2800u : 0x3c00u) | (w5 >> hi & 1u ? 0x28000000u : 0x3c000000u); }; // 2^-5 or 1
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    raw.ks[i] = hmul2(raw.ks[i], scale(g, 8 + g));
#pragma unroll
                    for (int h = 0; h < 2; h++) dv[h][i] = hmul2(dv[h][i], scale(16 + 8 * h + 2 * t, 17 + 8 * h + 2 * t));
                }
                if (lane == 0) sh.odd[ks][w] = make_uint4(w5, nan[0], nan[1], w5 | nan[0] | nan[1]);
            }
#pragma unroll
            for (int i = 0; i < NG; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t x[4];
                    unpack(raw.k[h][i], one, x);
                    const uint32_t dk = __byte_perm(raw.ks[i], 0, h ? 0x3232 : 0x1010);
                    sts128(k_at + ks * chunk_tile_bytes(HS) + h * 512 + i * (CHUNK_KEYS * 64), hmul2(x[0], dk), hmul2(x[1], dk), hmul2(x[2], dk), hmul2(x[3], dk));
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.k_full[ks]);
            if (++ks == CHUNK_K_STAGES) {
                ks = 0;
                k_phase ^= 1;
            }
            if (j + 1 < count) fetch(); // on its way while the values are converted
            if (j >= 2 && !__all_sync(0xffffffffu, bar_wait(&sh.v_free[b], ((j >> 1) - 1) & 1, &sh.bail))) break; // the products of tile j - 2 have read its values
#pragma unroll
            for (int i = 0; i < NG; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t x[4];
                    unpack(v[h][i], one, x);
                    // rows 32 i + 8 u + g: entries 32 i + 4 g + u
                    store_matrices((v_at + b * chunk_tile_bytes(HS) + i * 4096) ^ h * 16, hmul2(x[0], dv[h][i]), hmul2(x[1], dv[h][i]), hmul2(x[2], dv[h][i]), hmul2(x[3], dv[h][i]));
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.v_full[b]);
        }
    } else if (warp == CHUNK_ISSUER) {
        // ===== products =====
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(CHUNK_KEYS >> 3) << 17) | ((uint32_t)(CHUNK_ROWS >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t)(HS >> 3) << 17) | ((uint32_t)(CHUNK_ROWS >> 4) << 24);
        const uint32_t q = s32(sQ), lead = lane == 0;
        const auto passed = [&](const void *bar, unsigned parity) { return __all_sync(0xffffffffu, bar_wait<false>(bar, parity, &sh.bail)) != 0; };
        const auto scores = [&](int stage, int h) { // S = Q K^T
            const uint32_t k0 = s32(sK) + stage * chunk_tile_bytes(HS);
#pragma unroll
            for (int k = 0; k < HS / 16; k++)
                umma_ss(tS + h * CHUNK_KEYS, desc64(q + (k / 2) * (CHUNK_ROWS * 64) + (k % 2) * 32), desc64(k0 + (k / 2) * (CHUNK_KEYS * 64) + (k % 2) * 32), idesc_s, k > 0, lead);
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
            const uint32_t v0 = s32(sV) + h * chunk_tile_bytes(HS);
#pragma unroll
            for (int k = 0; k < CHUNK_KEYS / 16; k++) // O += P V
                umma_ts(tO + h * CHUNK_KEYS, tS + h * CHUNK_KEYS + (k / 4) * (CHUNK_KEYS / 2) + (k % 4) * 8, desc128(v0 + (k / 4) * (HS * 128) + (k % 4) * 32), idesc_o, j > 1 || k > 0, lead);
            umma_commit(&sh.v_free[h], lead);
            if (lead) *repeat = 0;
            __syncwarp();
            if (j + 2 < count) {
                if (!(ok = passed(&sh.k_full[ahead], phase))) break;
                fence_after();
                scores(ahead, h);
            } else umma_commit(&sh.s_full[h], lead);
            if (++stage == CHUNK_K_STAGES) stage = 0;
            if (++ahead == CHUNK_K_STAGES) {
                ahead = 0;
                phase ^= 1;
            }
        }
        // what is under way ends before the tensor memory goes: the warps of the rows have waited for it, or one of them has given up
        unsigned none = 0;
        umma_commit(&sh.drained, lead);
        if (!bar_wait(&sh.drained, 0, &none)) *reinterpret_cast<volatile unsigned *>(&sh.bail) = 1u;
    } else if (warp < CHUNK_SOFTMAX) {
        // ===== rows: two threads a stream, 64 positions of a tile a thread =====
        constexpr int PIECE = 16, COLUMNS = CHUNK_KEYS / 2;
        const int side = warp / 8, stream = warp / 4 % 2, r = tid % CHUNK_ROWS, token = token_of(r);
        const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16, row_s = tS + lanes + stream * CHUNK_KEYS + side * COLUMNS, row_o = tO + lanes + stream * CHUNK_KEYS;
        const float factor = sh.factor[r];
        unsigned met = 0;
        int j = stream - 2; // the tile
        const auto times32 = [](uint32_t (&x)[PIECE], uint32_t which) { // the low bits of `which`: whose numbers
            if (which & 0xffffu)
#pragma unroll
                for (int i = 0; i < PIECE; i++)
                    if (which >> i & 1u) x[i] = __float_as_uint(__uint_as_float(x[i]) * 32.0f);
        };
        const auto odds = [&](int q) -> const uint4 & { return sh.odd[j % CHUNK_K_STAGES][side * (CHUNK_RECORDS / 2) + q / PIECE]; }; // of the record of columns q on
        const auto meet = [&]() { // the two warps of a row; a wait with an end, as all here: one of them may have given up
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.pair[warp % 8]);
            return __all_sync(0xffffffffu, bar_wait(&sh.pair[warp % 8], met++ & 1, &sh.bail)) != 0;
        };
        int lo = 0, hi = 0, own = -1, seg = 0;
        if (token < tokens && sh.segment[token] >= 0) {
            own = sh.segment[token];
            visible(sh.pos[token], a.window, lo, hi);
        }
        float top = -CUDART_INF_F, l = 0.0f, sum = 0.0f; // the row's largest product so far; of this thread's positions the sum, and that of a tile that may yet be repeated
        bool ok = true, fresh = false;
        float base = 0.0f, ref = 0.0f; // top where there is one, times the factor
        int from = 0, to = 0, next = 0; // the tile's positions [from, to) are seen, counted from this thread's first; the segment's end
        const auto rows = [&](auto marked) {
        constexpr bool ODD = decltype(marked)::value; // (a body of its own: the other one keeps its registers)
        for (unsigned turn = 0; stream < count; turn++) {
            if (GIVE_UP && j + 2 >= count) {
                bar_wait(&sh.pair[warp % 8], met & 1, &sh.bail);
                break;
            }
            ok = __all_sync(0xffffffffu, bar_wait(&sh.s_full[stream], turn & 1, &sh.bail));
            if (!ok) break;
            fence_after();
            const bool repeat = *reinterpret_cast<volatile unsigned *>(&sh.repeat[stream]);
            if (!repeat) {
                l += sum;
                if ((j += 2) >= count) break;
                if (first + j >= next) {
                    while (sh.segments[seg].tiles <= first + j) seg++;
                    next = sh.segments[seg].tiles;
                    const int before = seg ? sh.segments[seg - 1].tiles : 0, key0 = (sh.segments[seg].begin + (first + j - before) * CHUNK_RECORDS) * BLOCK + side * COLUMNS;
                    from = own == seg ? lo - key0 : 0;
                    to = own == seg ? hi - key0 : 0;
                } else {
                    from -= 2 * CHUNK_KEYS;
                    to -= 2 * CHUNK_KEYS;
                }
                fresh = top == -CUDART_INF_F && max(from, -side * COLUMNS) < min(to, CHUNK_KEYS - side * COLUMNS); // the first that the row sees: no maximum yet
            }
            // One pass with the maximum as it stands.  It moves rarely, and a sum of more than 2^8 shows that it has to: the probabilities, which have taken the place of the scores, are
            // dropped, the scores come once more, and the tile's maximum is looked for first.  (A maximum of every tile in front of or beside the exponentials cost as much as they do.)
            const bool odd = ODD && __any_sync(0xffffffffu, odds(lane % (CHUNK_RECORDS / 2) * PIECE).w != 0u);
            const bool special = odd || __any_sync(0xffffffffu, repeat || fresh || from > 0 || to < COLUMNS || !(fabsf(ref) <= 65536.0f));
            if (special && __any_sync(0xffffffffu, repeat || fresh)) { // (the same for both warps of a row)
                float mx = -CUDART_INF_F;
#pragma unroll 1
                for (int q = 0; q < COLUMNS; q += PIECE) {
                    uint32_t x[PIECE];
                    tmem_ld16(row_s + q, x);
                    tmem_ld_wait();
                    if (odd) times32(x, odds(q).x);
#pragma unroll
                    for (int i = 0; i < PIECE; i++) mx = fmaxf(mx, i >= from - q && i < to - q ? __uint_as_float(x[i]) : -CUDART_INF_F);
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
                ref = base * factor;
            }
            // P takes the place of S: piece q of 16 scores is read before its 8 columns are written, [8 q, 8 q + 8)
            if (special && !__any_sync(0xffffffffu, max(from, 0) < min(to, COLUMNS))) { // other rows' tile
                const uint32_t p[PIECE / 2] = {};
                sum = 0.0f;
#pragma unroll 1
                for (int q = 0; q < COLUMNS / 2; q += PIECE / 2) tmem_st8(row_s + q, p);
            } else if (special && __any_sync(0xffffffffu, odd || from > 0 || to < COLUMNS || !(fabsf(ref) <= 65536.0f))) { // a border, entries outside FP16, or scores so large that their products and the maximum's round apart
                sum = 0.0f;
#pragma unroll 1
                for (int q = 0; q < COLUMNS; q += PIECE) {
                    uint32_t x[PIECE], p[PIECE / 2];
                    tmem_ld16(row_s + q, x);
                    tmem_ld_wait();
                    if (odd) times32(x, odds(q).x);
#pragma unroll
                    for (int i = 0; i < PIECE; i++) {
                        const float e = i >= from - q && i < to - q ? ex2((__uint_as_float(x[i]) - base) * factor) : 0.0f;
                        sum += e;
                        x[i] = __float_as_uint(e);
                    }
                    if (odd) {
                        const uint4 at = odds(q);
                        times32(x, at.x >> 16); // (at most 2^8 times that: FP16 holds it)
                        if (at.y | at.z) {
                            const int a = max(from - q, 0), b = min(to - q, PIECE);
                            const unsigned seen = a < b ? (1u << b) - (1u << a) : 0u, both = seen | seen << 16;
                            const unsigned groups = (at.y & both & 0xffffu ? 1u : 0u) | (at.y & both & 0xffff0000u ? 2u : 0u) | (at.z & both & 0xffffu ? 4u : 0u) | (at.z & both & 0xffff0000u ? 8u : 0u);
                            if (groups) atomicOr(&sh.nan[r], groups);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < PIECE / 2; i++) p[i] = pack_f16(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
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
                        p[i] = pack_f16(e0, e1);
                    }
                    tmem_st8(row_s + q * (PIECE / 2), p);
                }
                float a0, a1, b0, b1;
                unpack_f32x2(part[0], a0, a1);
                unpack_f32x2(part[1], b0, b1);
                sum = (a0 + a1) + (b0 + b1);
            }
            const bool over = __any_sync(0xffffffffu, !repeat && sum > 256.0f);
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (over) *reinterpret_cast<volatile unsigned *>(&sh.again[stream]) = 1u;
                bar_arrive(&sh.p_full[stream]);
            }
        }
        };
        if (__any_sync(0xffffffffu, sh.marked != 0u)) rows(std::true_type());
        else rows(std::false_type());
        sh.half_row[stream][side][r] = l;
        sh.top[stream][r] = top;
        fence_before();
    }
    __syncthreads();
    // ===== results: the streams are joined; a warp takes 32 rows and 32 entries =====
    if (warp < 4 * NG && sh.bail == 0u) {
        fence_after();
        const int q = warp / 4, r = warp % 4 * 32 + lane, token = token_of(r), row = token0 + token, head = kvh * mul + r - token * mul;
        const bool on = token < tokens && sh.slot[min(token, CHUNK_ROWS - 1)] >= 0;
        const float factor = sh.factor[r], t0 = sh.top[0][r], t1 = sh.top[1][r], top = fmaxf(t0, t1), base = top == -CUDART_INF_F ? 0.0f : top;
        const float a0 = t0 == base ? 1.0f : ex2((t0 - base) * factor), a1 = t1 == base ? 1.0f : ex2((t1 - base) * factor);
        const float l = a0 * (sh.half_row[0][0][r] + sh.half_row[0][1][r]) + a1 * (sh.half_row[1][0][r] + sh.half_row[1][1][r]);
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 32; i++) o[i] = 0u;
        for (int h = 0; h < min(count, 2); h++) { // (a stream without tiles has no sums)
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
                uint32_t x[16];
                tmem_ld16(tO + ((uint32_t)(warp % 4 * 32) << 16) + h * CHUNK_KEYS + q * 32 + i, x);
                tmem_ld_wait();
#pragma unroll
                for (int u = 0; u < 16; u++) o[i + u] = __float_as_uint(fmaf(h ? a1 : a0, __uint_as_float(x[u]), __uint_as_float(o[i + u])));
            }
        }
        if (sh.nan[r] >> q & 1u)
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = 0x7fffffffu;
        if (c.splits > 1) { // parts go through shared memory, where the queries were: 64 bytes of a row at a time in place of 4 (the rows' starts are 8-byte aligned)
            const long long part = on ? (((long long)row * a.heads + head) * c.splits + split) * (HS + 2) : -1;
            if (on && q == 0) { a.work[part] = top * factor; a.work[part + 1] = l; }
            const uint32_t at = s32(sQ) + warp * 2048;
#pragma unroll 1
            for (int e = 0; e < 32; e += 16) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; i++) // entries e + 4 i .. + 3: entry x of the group is column 8 (x % 4) + x / 4
                    sts128(at + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4), e ? o[4 + i] : o[i], e ? o[12 + i] : o[8 + i], e ? o[20 + i] : o[16 + i], e ? o[28 + i] : o[24 + i]);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int k = 4 * i + lane / 8;
                    float2 x;
                    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at + k * 64 + ((lane % 8 / 2 ^ (k >> 1 & 3)) << 4) + (lane & 1) * 8) : "memory");
                    const long long to = __shfl_sync(0xffffffffu, part, k);
                    if (to >= 0) *reinterpret_cast<float2 *>(a.work + to + 2 + q * 32 + e + lane % 8 * 2) = x;
                }
            }
        } else if (on) {
            int lo, hi;
            visible(sh.pos[token], a.window, lo, hi);
            const float inv = hi > lo ? 1.0f / l : 0.0f;
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float v0 = __uint_as_float(o[8 * (2 * i % 4) + 2 * i / 4]) * inv, v1 = __uint_as_float(o[8 * ((2 * i + 1) % 4) + (2 * i + 1) / 4]) * inv;
                if (a.out_type == B200_GGML_F16) y[i] = pack_f16(v0, v1);
                else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
                    y[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            uint16_t *out = (uint16_t *)a.out + row * a.ldo + (size_t)head * HS + q * 32;
            if (c.vec_out)
#pragma unroll
                for (int i = 0; i < 4; i++) reinterpret_cast<uint4 *>(out)[i] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
            else
#pragma unroll
                for (int i = 0; i < 32; i++) out[i] = (uint16_t)(y[i / 2] >> (i & 1) * 16);
        }
        fence_before();
    }
    __syncthreads();
    if (tid == 0 && sh.bail != 0u) *reinterpret_cast<volatile unsigned *>(c.error) = a.kv.odd[a.kv.slots] = 1u;
    if (warp == CHUNK_SOFTMAX) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

} // namespace kv4
