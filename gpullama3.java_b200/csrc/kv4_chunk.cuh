// kv4_chunk.cuh -- attention of prompt chunks over the 4-bit cache on the 5th-generation tensor cores, with 16-bit results.
//
// A CTA takes 128 rows (tokens x query heads of one key/value head) and runs through the positions that any of them sees, 128 at a time:
//   warps 8-23  turn a tile's records (half a record a warp) into FP16 operands in shared memory: keys [position][entry], values transposed [entry][position], both K-major
//   one thread  issues S = Q K^T (two accumulators in TMEM, so that a tile's product runs while the rows work on the one before) and O += P V, with P read from TMEM
//   warps 0-7   half a row a thread: exponentials, P as FP16 into TMEM; O is scaled where a row's maximum has grown by too much, which is rare
// Per tile of heads of 128: 1024 cycles of products (8192 FLOP a cycle), 1024 of exponentials (16 a cycle), about 1200 issue slots a scheduler: all three side by side.  What they
// wait for is latency: with 4 and 8 warps in place of 8 and 16 a tile took 3000 cycles, 2000 of them in a row's exponentials and as many in a record's conversion.
// Rounding: queries (times a power of two), keys, values and probabilities are FP16 operands, sums are FP32.  A value's NaN, or one outside FP16, is moved into its key, so that it
// reaches the rows that see the position and no other (0 * NaN in the product would reach them all).
//
// Rows of a tile may belong to several slots and stand in any order: a run of tokens of one slot is a segment, the tiles of all segments are one list, and a row masks what is not its own.
// Every wait is bounded: after two seconds the CTA gives up, writes the cache's error word, waits for its products under way and frees its tensor memory.
#pragma once
#include <type_traits>

#include "kv4.cuh"

namespace kv4 {

constexpr int CHUNK_ROWS = 128, CHUNK_KEYS = 128, CHUNK_RECORDS = CHUNK_KEYS / BLOCK;
constexpr int CHUNK_SOFTMAX = 8, CHUNK_DEQUANT = 16, CHUNK_ISSUER = CHUNK_SOFTMAX + CHUNK_DEQUANT, CHUNK_THREADS = (CHUNK_ISSUER + 1) * 32; // warps of each kind
__host__ __device__ constexpr int chunk_q_bytes(int hs) { return groups(hs) * CHUNK_ROWS * 64; }
__host__ __device__ constexpr int chunk_stage_bytes(int hs) { return groups(hs) * CHUNK_KEYS * 64 + hs * CHUNK_KEYS * 2; }

struct Segment { // a run of tokens of one slot and the records that any of them sees
    int slot, begin, end, tiles; // records [begin, end); tiles of all segments up to and with this one
};
struct ChunkSmem { // behind the operands
    unsigned long long k_full[2], v_full[2], free[2], s_full[2], s_empty[2], p_full[2], pair[4], drained;
    unsigned tmem, bail;
    int n_segments, single;
    int slot[CHUNK_ROWS], pos[CHUNK_ROWS], segment[CHUNK_ROWS]; // by token
    float factor[CHUNK_ROWS];                                   // by row: what turns a product into a score in units of log2
    float half_row[2][CHUNK_ROWS];                              // what the two threads of a row tell each other
    int again[2][CHUNK_SOFTMAX];                                // by tile and warp: a row's maximum has to move
    Segment segments[CHUNK_ROWS];
};
__host__ __device__ constexpr size_t chunk_smem_bytes(int hs) { return 1024 + chunk_q_bytes(hs) + 2 * chunk_stage_bytes(hs) + sizeof(ChunkSmem); }

__device__ __forceinline__ uint32_t s32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(const void *bar, unsigned n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(bar)), "r"(n)); }
__device__ __forceinline__ void bar_arrive(const void *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(bar)) : "memory"); }
__device__ __forceinline__ bool bar_wait(const void *bar, unsigned parity, unsigned *bail) { // false: given up
    const uint32_t b = s32(bar);
    unsigned long long began = 0;
    for (unsigned i = 1;; i++) {
        unsigned done;
        asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}" : "=r"(done) : "r"(b), "r"(parity) : "memory");
        if (done) return true;
        if ((i & 255u) == 0u) {
            if (*reinterpret_cast<volatile unsigned *>(bail)) return false;
            const unsigned long long now = gtime_ns();
            if (!began) began = now;
            else if (now - began > 2000000000ull) {
                *reinterpret_cast<volatile unsigned *>(bail) = 1u;
                return false;
            }
        }
    }
}
// K-major operand descriptors: start >> 4 | 1 << 16 | 8 rows >> 4 << 32 | version 1 << 46 | swizzle (2: rows of 128 bytes, 4: rows of 64) << 61
__device__ __forceinline__ uint64_t desc128(uint32_t a) { return (uint64_t)((a & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61); }
__device__ __forceinline__ uint64_t desc64(uint32_t a) { return (uint64_t)((a & 0x3ffffu) >> 4) | (1ull << 16) | (32ull << 32) | (1ull << 46) | (4ull << 61); }
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) { // the first operand from TMEM
    asm volatile("{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void umma_commit(const void *bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
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
__device__ __forceinline__ void sts32(uint32_t a, uint32_t x) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// What a dequantising lane holds of half a record: codes, the key scales of positions g and g + 8, the value scales of positions 2 t, 2 t + 8 and 2 t + 1, 2 t + 9.
template <int HS> struct Raw {
    static constexpr int NG = groups(HS), VW = vec_words(HS);
    uint32_t k[NG], v[NG], ks[NG], vs[2][NG];
    __device__ __forceinline__ void load(const unsigned char *rec, int half, int lane) {
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
            get(w + word_of<HS>(half, lane, c * VW), k + c * VW);
            get(w + 2 * HS + word_of<HS>(half, lane, c * VW), v + c * VW);
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

template <int HS> __global__ void __launch_bounds__(CHUNK_THREADS, 1) k_chunk(const Chunk c) {
    constexpr int NG = groups(HS);
    extern __shared__ unsigned char raw_smem[];
    unsigned char *smem = raw_smem + (-s32(raw_smem) & 1023u); // the operands' swizzle counts from 1024-byte boundaries
    unsigned char *sQ = smem, *stages = smem + chunk_q_bytes(HS);
    ChunkSmem &sh = *reinterpret_cast<ChunkSmem *>(stages + 2 * chunk_stage_bytes(HS));
    const Step &a = c.step;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.kv.kv_heads, mul = a.heads / G;
    const int n_tiles = (a.rows.n + c.tokens - 1) / c.tokens;
    const int split = blockIdx.x % c.splits, kvh = blockIdx.x / c.splits % G, tile = n_tiles - 1 - blockIdx.x / c.splits / G; // the last tokens, which see most, first
    const int token0 = tile * c.tokens, tokens = min(c.tokens, a.rows.n - token0);

    pdl_wait();
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            bar_init(&sh.k_full[i], CHUNK_DEQUANT);
            bar_init(&sh.v_full[i], CHUNK_DEQUANT);
            bar_init(&sh.free[i], 1);
            bar_init(&sh.s_full[i], 1);
            bar_init(&sh.s_empty[i], CHUNK_SOFTMAX);
            bar_init(&sh.p_full[i], CHUNK_SOFTMAX);
        }
        for (int i = 0; i < 4; i++) bar_init(&sh.pair[i], 2);
        bar_init(&sh.drained, 1);
        sh.bail = 0;
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
        }
        sh.slot[tid] = slot;
        sh.pos[tid] = pos;
        sh.segment[tid] = -1;
    }
    // queries: a row a warp, all of a warp's rows under way at once
    constexpr int WARPS = CHUNK_THREADS / 32, QROWS = (CHUNK_ROWS + WARPS - 1) / WARPS;
    float4 x[QROWS]; // entries 4 lane .. + 3
#pragma unroll
    for (int i = 0; i < QROWS; i++) {
        const int r = warp + i * WARPS, token = r / mul;
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (token < tokens && r < CHUNK_ROWS && lane * 4 < HS) {
            const float *q = a.q + (long long)(token0 + token) * a.ldq + (size_t)(kvh * mul + r % mul) * HS + lane * 4;
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
    const uint32_t tmem = sh.tmem, tS = tmem, tP = tmem + 256, tO = tmem + 384;
    const int total = sh.n_segments ? sh.segments[sh.n_segments - 1].tiles : 0;
    const int first = (int)((long long)total * split / c.splits), last = (int)((long long)total * (split + 1) / c.splits), count = last - first;

    if (warp >= CHUNK_SOFTMAX && warp < CHUNK_ISSUER) {
        // ===== records -> FP16 operands =====
        const int d = warp - CHUNK_SOFTMAX, w = d / 2, half = d % 2, g = lane >> 2, t = lane & 3;
        const uint32_t one = magic();
        int seg = 0, ahead = 0, block = 0, stop = 0, behind = 0; // tiles left in the segment, this warp's record in the next one, the segment's end; raw is a record behind it
        if (count > 0) {
            while (sh.segments[seg].tiles <= first) seg++;
            const int before = seg ? sh.segments[seg - 1].tiles : 0;
            ahead = sh.segments[seg].tiles - first;
            block = sh.segments[seg].begin + (first - before) * CHUNK_RECORDS + w;
            stop = sh.segments[seg].end;
        }
        auto fetch = [&](Raw<HS> &to) { // this warp's half record of the list's next tile; behind the segment's end its last one, whose values then count as zeros
            if (ahead == 0) {
                seg++;
                ahead = sh.segments[seg].tiles - sh.segments[seg - 1].tiles;
                block = sh.segments[seg].begin + w;
                stop = sh.segments[seg].end;
            }
            behind = block >= stop;
            to.load(record<HS>(a.kv, sh.segments[seg].slot, kvh, min(block, stop - 1)), half, lane);
            ahead--;
            block += CHUNK_RECORDS;
        };
        // row 16 w + 8 half + g of the keys; positions 16 w + 8 half + 2 t, + 1 of the values: 16-byte chunk 2 (w % 4) + half of the rows of 64 positions
        const uint32_t k_at = s32(stages) + (w * 16 + half * 8 + g) * 64 + ((t ^ (g >> 1 & 3)) << 4);
        const uint32_t v_at = s32(stages) + NG * CHUNK_KEYS * 64 + (w / 4) * (HS * 128) + g * 128 + (((w % 4 * 2 + half) ^ g) << 4) + t * 4;
        const uint32_t k_perm = half ? 0x3232 : 0x1010, v_perm = half ? 0x7632 : 0x5410;
        struct Held { // a half record's values, until the product two tiles before them has read its own
            uint32_t v[NG], d[NG]; // codes, scales of positions 8 half + 2 t and + 1
        };
        auto keys = [&](int j, Raw<HS> &now, Held &held) {
            // a value scale that FP16 products do not hold (or a NaN) is moved into the keys: such positions get no value and a NaN key
            __half2 widest;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                held.v[i] = now.v[i];
                held.d[i] = __byte_perm(now.vs[0][i], now.vs[1][i], v_perm);
                const __half2 x = __habs2(*reinterpret_cast<const __half2 *>(&held.d[i]));
                widest = i ? __hmax2_nan(widest, x) : x;
            }
            const uint32_t wide = *reinterpret_cast<const uint32_t *>(&widest);
            if (behind)
#pragma unroll
                for (int i = 0; i < NG; i++) held.d[i] = 0u;
            if (__any_sync(0xffffffffu, (0xeffeeffeu - wide & 0x80008000u) != 0x80008000u)) { // a half above 0x6ffe: 8 d up to 65504
                uint32_t bad = ((wide & 0xffffu) > 0x6ffeu ? 1u << (2 * t) : 0u) | (wide >> 16 > 0x6ffeu ? 2u << (2 * t) : 0u); // by position of the half
                bad = __reduce_or_sync(0xffffffffu, bad);
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    if (bad >> (2 * t) & 1u) held.d[i] &= 0xffff0000u;
                    if (bad >> (2 * t + 1) & 1u) held.d[i] &= 0x0000ffffu;
                    if (bad >> g & 1u) now.ks[i] = 0x7fff7fffu;
                }
            }
            const int b = j & 1;
            if (j >= 2 && !__all_sync(0xffffffffu, bar_wait(&sh.s_full[b], ((j >> 1) - 1) & 1, &sh.bail))) return false; // the product of tile j - 2 has read its keys
            const uint32_t at = k_at + b * chunk_stage_bytes(HS);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                uint32_t x[4];
                unpack(now.k[i], one, x);
                const uint32_t dk = __byte_perm(now.ks[i], 0, k_perm);
                sts128(at + i * (CHUNK_KEYS * 64), hmul2(x[0], dk), hmul2(x[1], dk), hmul2(x[2], dk), hmul2(x[3], dk));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.k_full[b]);
            return true;
        };
        auto values = [&](int j, const Held &held) {
            const int b = j & 1;
            if (j >= 2 && !__all_sync(0xffffffffu, bar_wait(&sh.free[b], ((j >> 1) - 1) & 1, &sh.bail))) return false; // the product of tile j - 2 has read its values
            const uint32_t at = v_at + b * chunk_stage_bytes(HS);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                uint32_t x[4];
                unpack(held.v[i], one, x);
#pragma unroll
                for (int u = 0; u < 4; u++) sts32(at + (i * 32 + u * 8) * 128, hmul2(x[u], held.d[i])); // row 32 i + 8 u + g: entry 32 i + 4 g + u
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.v_full[b]);
            return true;
        };
        // Keys run a tile ahead of the values, which wait for the rows; the next record is asked for when this one's registers have been read, not before: loads share their
        // scoreboards, and a wait for the older ones would be one for both (800 cycles a tile).
        Raw<HS> raw;
        Held even, odd;
        bool ok = true;
        if (count > 0) {
            fetch(raw);
            ok = keys(0, raw, even);
            if (count > 1) fetch(raw);
        }
        for (int j = 0; j < count && ok; j += 2) {
            if (j + 1 < count) {
                if (!(ok = keys(j + 1, raw, odd))) break;
                if (j + 2 < count) fetch(raw);
            }
            if (!(ok = values(j, even)) || j + 1 >= count) break;
            if (j + 2 < count) {
                if (!(ok = keys(j + 2, raw, even))) break;
                if (j + 3 < count) fetch(raw);
            }
            ok = values(j + 1, odd);
        }
    } else if (warp == CHUNK_ISSUER && lane == 0) {
        // ===== products =====
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(CHUNK_KEYS >> 3) << 17) | ((uint32_t)(CHUNK_ROWS >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t)(HS >> 3) << 17) | ((uint32_t)(CHUNK_ROWS >> 4) << 24);
        const uint32_t q = s32(sQ), st = s32(stages);
        auto product = [&](int j) { // O += P V of tile j
            const int b = j & 1;
            if (!bar_wait(&sh.v_full[b], j >> 1 & 1, &sh.bail) || !bar_wait(&sh.p_full[b], j >> 1 & 1, &sh.bail)) return false;
            fence_after();
            const uint32_t sV = st + b * chunk_stage_bytes(HS) + NG * CHUNK_KEYS * 64;
#pragma unroll
            for (int k = 0; k < CHUNK_KEYS / 16; k++) umma_ts(tO, tP + b * 64 + k * 8, desc128(sV + (k / 4) * (HS * 128) + (k % 4) * 32), idesc_o, j > 0 || k > 0);
            umma_commit(&sh.free[b]);
            return true;
        };
        bool ok = true;
        for (int j = 0; j < count && ok; j++) {
            const int b = j & 1;
            ok = bar_wait(&sh.k_full[b], j >> 1 & 1, &sh.bail) && (j < 2 || bar_wait(&sh.s_empty[b], ((j >> 1) - 1) & 1, &sh.bail));
            if (!ok) break;
            fence_after();
            const uint32_t sK = st + b * chunk_stage_bytes(HS);
#pragma unroll
            for (int k = 0; k < HS / 16; k++) umma_ss(tS + b * 128, desc64(q + (k / 2) * (CHUNK_ROWS * 64) + (k % 2) * 32), desc64(sK + (k / 2) * (CHUNK_KEYS * 64) + (k % 2) * 32), idesc_s, k > 0);
            umma_commit(&sh.s_full[b]);
            if (j > 0) ok = product(j - 1);
        }
        if (ok && count > 0) ok = product(count - 1);
        if (!ok) { // given up: what is under way ends before the tensor memory goes
            unsigned none = 0;
            umma_commit(&sh.drained);
            bar_wait(&sh.drained, 0, &none);
            if (c.error) *reinterpret_cast<volatile unsigned *>(c.error) = 1u;
        }
    } else if (warp < CHUNK_SOFTMAX) {
        // ===== rows: warps w and w + 4 share 32 of them, 64 positions of a tile and half of the entries each =====
        constexpr int COLUMNS = CHUNK_KEYS / 2, PIECE = 16;
        const int side = warp / 4, r = warp % 4 * 32 + lane, token = r / mul;
        const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16; // this warp's part of the tensor memory
        const int group0 = side ? (NG + 1) / 2 : 0, group1 = side ? NG : (NG + 1) / 2;
        const float factor = sh.factor[r];
        unsigned met = 0;
        const auto meet = [&]() { // the two warps of a row; a wait with an end, as all here: one of them may have given up
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.pair[warp % 4]);
            return __all_sync(0xffffffffu, bar_wait(&sh.pair[warp % 4], met++ & 1, &sh.bail)) != 0;
        };
        int lo = 0, hi = 0, own = -1, seg = 0;
        if (token < tokens && sh.segment[token] >= 0) {
            own = sh.segment[token];
            visible(sh.pos[token], a.window, lo, hi);
        }
        while (seg < sh.n_segments && sh.segments[seg].tiles <= first) seg++;
        float m = -CUDART_INF_F, l = 0.0f; // of the row; of this thread's positions
        bool ok = true;
        for (int j = 0; j < count; j++) {
            const int b = j & 1;
            while (sh.segments[seg].tiles <= first + j) seg++;
            const int before = seg ? sh.segments[seg - 1].tiles : 0, key0 = (sh.segments[seg].begin + (first + j - before) * CHUNK_RECORDS) * BLOCK;
            int from = lo - key0, to = hi - key0; // the tile's positions [from, to) are seen
            if (own != seg) from = to = 0;
            const bool fresh = m == -CUDART_INF_F && max(from, 0) < min(to, CHUNK_KEYS); // the first that the row sees
            from -= side * COLUMNS;
            to -= side * COLUMNS;
            const bool mask = __any_sync(0xffffffffu, from > 0 || to < COLUMNS);
            ok = __all_sync(0xffffffffu, bar_wait(&sh.s_full[b], j >> 1 & 1, &sh.bail));
            if (!ok) break;
            fence_after();
            if (j >= 2) { // P's buffer: its last product has read it
                ok = __all_sync(0xffffffffu, bar_wait(&sh.free[b], ((j >> 1) - 1) & 1, &sh.bail));
                if (!ok) break;
            }
            const uint32_t row_s = tS + lanes + b * CHUNK_KEYS + side * COLUMNS, row_p = tP + lanes + b * (CHUNK_KEYS / 2) + side * (COLUMNS / 2);
            // One pass with the maximum as it stands.  It moves rarely, and a sum of more than 2^8 shows that it has to: then the tile's maximum is looked for and the pass made again.
            // (A maximum of every tile in front of or beside the exponentials cost as much as they do.)
            float sum;
            const auto exponentials_of = [&](auto masked, float ref) {
                const unsigned long long factor2 = pack_f32x2(factor, factor), ref2 = pack_f32x2(-ref, -ref);
                unsigned long long part[2] = {0ull, 0ull};
                uint32_t s[2][PIECE];
                tmem_ld16(row_s, s[0]);
#pragma unroll
                for (int q = 0; q < COLUMNS / PIECE; q++) {
                    uint32_t(&x)[PIECE] = s[q & 1];
                    tmem_ld_wait();
                    if (q + 1 < COLUMNS / PIECE) tmem_ld16(row_s + (q + 1) * PIECE, s[q + 1 & 1]);
                    if constexpr (decltype(masked)::value)
#pragma unroll
                        for (int i = 0; i < PIECE; i++)
                            if (!(q * PIECE + i >= from && q * PIECE + i < to)) x[i] = 0xff800000u;
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
                    tmem_st8(row_p + q * (PIECE / 2), p);
                }
                float a0, a1, b0, b1;
                unpack_f32x2(part[0], a0, a1);
                unpack_f32x2(part[1], b0, b1);
                sum = (a0 + a1) + (b0 + b1);
            };
            const auto exponentials = [&](float ref) {
                if (mask) exponentials_of(std::true_type(), ref);
                else exponentials_of(std::false_type(), ref);
            };
            exponentials(m == -CUDART_INF_F ? 0.0f : m);
            const bool again = __any_sync(0xffffffffu, fresh || sum > 256.0f);
            if (lane == 0) sh.again[b][warp] = again;
            ok = meet();
            if (!ok) break;
            if (again || sh.again[b][warp ^ 4]) {
                float mx = -CUDART_INF_F;
#pragma unroll 1
                for (int q = 0; q < COLUMNS / PIECE; q++) {
                    uint32_t x[PIECE];
                    tmem_ld16(row_s + q * PIECE, x);
                    tmem_ld_wait();
                    const int lo_q = from - q * PIECE, hi_q = to - q * PIECE;
#pragma unroll
                    for (int i = 0; i < PIECE; i++) mx = fmaxf(mx, i >= lo_q && i < hi_q ? __uint_as_float(x[i]) : -CUDART_INF_F);
                }
                sh.half_row[side][r] = mx;
                ok = meet();
                if (!ok) break;
                mx = fmaxf(mx, sh.half_row[side ^ 1][r]);
                const float grown = fmaxf(m, mx * factor), alpha = m == grown ? 1.0f : ex2(m - grown);
                m = grown;
                l *= alpha;
                if (j > 0) {
                    ok = __all_sync(0xffffffffu, bar_wait(&sh.free[b ^ 1], (j - 1) >> 1 & 1, &sh.bail));
                    if (!ok) break;
                    fence_after();
                    tmem_st_wait();
#pragma unroll 1
                    for (int q = group0 * 2; q < group1 * 2; q++) {
                        uint32_t o[PIECE];
                        tmem_ld16(tO + lanes + q * PIECE, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < PIECE; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st16(tO + lanes + q * PIECE, o);
                    }
                }
                exponentials(m == -CUDART_INF_F ? 0.0f : m);
            }
            l += sum;
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(&sh.s_empty[b]);
                bar_arrive(&sh.p_full[b]);
            }
        }
        if (ok && count > 0) ok = __all_sync(0xffffffffu, bar_wait(&sh.free[(count - 1) & 1], (count - 1) >> 1 & 1, &sh.bail));
        fence_after();
        if (ok) {
            sh.half_row[side][r] = l;
            ok = meet();
            l += sh.half_row[side ^ 1][r];
        }
        const bool on = token < tokens && sh.slot[min(token, CHUNK_ROWS - 1)] >= 0, some = hi > lo;
        const int row = token0 + token, head = kvh * mul + r % mul;
        const float inv = 1.0f / l;
#pragma unroll 1
        for (int q = group0; q < group1 && ok; q++) {
            uint32_t o[32];
            __syncwarp();
            if (count > 0) {
                tmem_ld32(tO + lanes + q * 32, o);
                tmem_ld_wait();
            } else
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = 0u;
            if (on && c.splits > 1) {
                float *w = a.work + (((size_t)row * a.heads + head) * c.splits + split) * (HS + 2);
                if (q == 0) { w[0] = m; w[1] = l; }
#pragma unroll
                for (int i = 0; i < 32; i++) w[2 + q * 32 + i] = __uint_as_float(o[8 * (i % 4) + i / 4]); // entry i of the group is column 8 (i % 4) + i / 4
            } else if (on) {
                uint32_t y[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float v0 = some ? __uint_as_float(o[8 * (2 * i % 4) + 2 * i / 4]) * inv : 0.0f, v1 = some ? __uint_as_float(o[8 * ((2 * i + 1) % 4) + (2 * i + 1) / 4]) * inv : 0.0f;
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
        }
        fence_before();
    }
    __syncthreads();
    if (warp == CHUNK_SOFTMAX) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

} // namespace kv4
