// kv4.cuh -- a key/value cache of 4-bit codes: append (head norms, rotation and quantisation in one pass), read-back, and the attention of single query rows over it.
//
// A group is 32 neighbouring entries of a head: a scale d (FP16) and codes c of 4 bits, value d * (c - 8).  m = the group's entry of largest magnitude (the first of equal ones),
// d = f16(m / -8), c = clamp(rint(x / d) + 8, 0, 15): m itself lands on an end of the range whatever its sign.  A group with an infinity or a NaN is stored with a NaN scale.
//
// Memory: [slot][key/value head][block of 16 positions] records of 18 * HS bytes, so that any run of positions of a head is ONE contiguous stretch:
//   key codes    [half: positions 0-7, 8-15][words of a lane / VW][lane = 4 g + t][VW words]: lane (g, t) holds position 8 * half + g, entries 32 grp + 8 t .. + 7 in word grp
//   value codes  the same order; lane (g, t) holds positions 8 * half + 2 t, + 1 (low and high half of a word) and entries 32 grp + 4 g .. + 3
//   key scales   [g][grp] words of two halves: positions g and g + 8; value scales likewise
// These are the operands of mma.m16n8k16 as its lanes want them: a lane reads its words in one vector load without bank conflicts, and a word's eight codes are four register pairs.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace kv4 {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int GROUP = 32, BLOCK = 16; // entries of a group, positions of a record
__host__ __device__ constexpr int groups(int hs) { return hs / GROUP; }
__host__ __device__ constexpr int vec_words(int hs) { return groups(hs) > 4 ? 4 : groups(hs); } // words that a lane loads at a time
__host__ __device__ constexpr int record_bytes(int hs) { return 18 * hs; }

struct View {
    unsigned char *base;
    unsigned *odd; // by slot: has it taken a group whose scale is beyond KV4_ODD or NaN (for as long as the cache is not reset); behind the slots: has a chunk's attention given up a wait
    int slots, context, blocks, kv_heads; // blocks of a head and slot
};
constexpr unsigned KV4_ODD = 0x6ffe; // FP16 bits of 8184: entries of up to 8 times a larger scale may lie outside FP16
struct Rows { // row r stands at position `positions ? positions[r] : start + r` of slot `slots ? slots[r] : slot`
    const int *positions, *slots;
    int n, start, slot;
    __device__ __forceinline__ int position(int r) const { return positions ? positions[r] : start + r; }
    __device__ __forceinline__ int slot_of(int r) const { return slots ? slots[r] : slot; }
};

template <int HS> __device__ __forceinline__ unsigned char *record(const View &kv, int slot, int head, int block) {
    return kv.base + (((size_t)slot * kv.kv_heads + head) * kv.blocks + block) * record_bytes(HS);
}
// Index of a lane's word `grp` in the codes of a record's half.
template <int HS> __device__ __forceinline__ int word_of(int half, int lane, int grp) {
    constexpr int NG = groups(HS), VW = vec_words(HS);
    return half * 32 * NG + (grp / VW) * 32 * VW + lane * VW + grp % VW;
}

__device__ __forceinline__ float load_f32(const float *p) { return *p; }
__device__ __forceinline__ void load8(const float *p, float (&x)[8], bool vec) {
    if (vec) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
}
__device__ __forceinline__ float2 to_f32x2(uint32_t w, const __half *) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 to_f32x2(uint32_t w, const bf16 *) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8], bool vec) {
    if (vec) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = to_f32x2(v[i], p);
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(p[i]);
}

// ---- append ---------------------------------------------------------------------------------------------------------------------------------------------------
struct Append {
    View kv;
    Rows rows;
    const void *q, *k, *v;
    long long ldq, ldk, ldv, ldo; // entries between rows
    int heads;                    // query heads; 0: none
    int interleaved, vec;         // vec: every row starts on a 16-byte boundary
    const float *q_norm, *k_norm, *cos, *sin; // norms and tables: null where there is none
    float eps;
    float *q_out;
};

// 4-bit codes of a lane's 8 entries; the four lanes of a group hold its 32.
__device__ __forceinline__ void quantize8(const float (&x)[8], unsigned lanes, __half &scale, int (&c)[8]) {
    float top = x[0];
    bool bad = !(fabsf(x[0]) < CUDART_INF_F);
#pragma unroll
    for (int i = 1; i < 8; i++) {
        if (fabsf(x[i]) > fabsf(top)) top = x[i];
        bad |= !(fabsf(x[i]) < CUDART_INF_F);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float other = __shfl_xor_sync(lanes, top, o);
        const bool lower = (threadIdx.x & o) != 0; // the other lane's entries stand in front of this one's
        if (fabsf(other) > fabsf(top) || (fabsf(other) == fabsf(top) && lower)) top = other;
        bad |= (bool)__shfl_xor_sync(lanes, (int)bad, o);
    }
    scale = bad ? __ushort_as_half(0x7fff) : __float2half_rn(fminf(fmaxf(top * -0.125f, -65504.0f), 65504.0f));
    const float d = __half2float(scale);
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = bad || d == 0.0f ? 8 : (int)fminf(fmaxf(rintf(__fdiv_rn(x[i], d)), -8.0f), 7.0f) + 8;
}

// Lanes of a head: 8 entries each, so that pairs of neighbours lie in a lane, pairs half a head apart in lanes half the head's lanes apart, and a group in four lanes.
// A segment of WIDTH lanes (a power of two) serves one head, 32 / WIDTH heads a warp.  Bytes are its floor: 512 rows of (32 + 2 * 8) heads of 128 with norms and
// rotation read 12.6 MB and write 9.0, 3.8 us; it takes 11.5 (1.12 TB/s), with the call 16.4.  1536 CTAs at 8 an SM are 1.3 waves of warps that
// load, reduce, normalise, turn, quantise and store one after the other: per issued instruction 7.4 wait for a load, 2.7 for a fixed latency, 2.6 for shuffles; codes leave in 2 and 4 bytes.
// (Tables asked for in front of the norm, which they do not need: more registers, 18-19 us.)
template <int HS, typename T> __global__ void __launch_bounds__(256) k_append(const Append a) {
    constexpr int L = HS / 8, WIDTH = L == 4 ? 4 : L == 8 ? 8 : L <= 16 ? 16 : 32, PER_WARP = 32 / WIDTH;
    pdl_wait();
    const int lane = threadIdx.x & 31, li = lane & (WIDTH - 1), G = a.kv.kv_heads, total = a.heads + 2 * G;
    const long long item = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * PER_WARP + lane / WIDTH;
    const int row = (int)(item / total), which = (int)(item % total);
    int pos = 0, slot = -1;
    if (row < a.rows.n) { pos = a.rows.position(row); slot = a.rows.slot_of(row); }
    const bool on = row < a.rows.n && pos >= 0 && pos < a.kv.context && slot >= 0 && slot < a.kv.slots, mine = on && li < L;
    if (!__any_sync(0xffffffffu, on)) return; // (a whole warp: the shuffles below take every lane)
    const bool is_q = which < a.heads, is_v = which >= a.heads + G;
    const int head = is_q ? which : is_v ? which - a.heads - G : which - a.heads;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    if (mine) {
        const T *src = is_q ? (const T *)a.q + row * a.ldq : is_v ? (const T *)a.v + row * a.ldv : (const T *)a.k + row * a.ldk;
        load8(src + head * HS + li * 8, x, a.vec);
    }
    const float *norm = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    { // mean of squares in 64 bits: one rounding to FP32, whatever the order of the sum
        double ss = 0.0;
        if (a.q_norm || a.k_norm) {
#pragma unroll
            for (int i = 0; i < 8; i++) ss += (double)x[i] * (double)x[i];
#pragma unroll
            for (int o = WIDTH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (norm && mine) {
            const float s = (float)rsqrt(ss * (1.0 / HS) + (double)a.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = norm[li * 8 + i] * (s * x[i]);
        }
    }
    if (a.cos) {
        const float *cs = a.cos + (size_t)pos * (HS / 2), *sn = a.sin + (size_t)pos * (HS / 2);
        if (a.interleaved) {
            if (mine && !is_v)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float c = cs[li * 4 + i], s = sn[li * 4 + i], u = x[2 * i], w = x[2 * i + 1];
                    x[2 * i] = u * c - w * s;
                    x[2 * i + 1] = u * s + w * c;
                }
        } else {
            const bool low = li < L / 2;
            const int partner = lane - li + (low ? li + L / 2 : li < L ? li - L / 2 : li);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], partner);
            if (mine && !is_v)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int at = (low ? li : li - L / 2) * 8 + i;
                    const float c = cs[at], s = sn[at];
                    x[i] = low ? x[i] * c - y[i] * s : y[i] * s + x[i] * c;
                }
        }
    }
    if (is_q) {
        if (mine) {
            float *o = a.q_out + row * a.ldo + head * HS + li * 8;
            if (a.vec) {
                *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4 *>(o + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = x[i];
        }
    }
    if (!__any_sync(0xffffffffu, mine && !is_q)) return; // (two thirds of the warps of a grouped model hold queries alone)
    __half scale;
    int c[8];
    quantize8(x, 0xffffffffu, scale, c);
    if (!mine || is_q) return;
    unsigned char *rec = record<HS>(a.kv, slot, head, pos / BLOCK);
    const int in = pos % BLOCK, half = in >> 3, grp = li >> 2, t = li & 3;
    if (!is_v) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) w |= (uint32_t)c[i] << (4 * (i >> 1) + 16 * (i & 1));
        reinterpret_cast<uint32_t *>(rec)[word_of<HS>(half, 4 * (in & 7) + t, grp)] = w;
    } else {
        uint16_t *codes = reinterpret_cast<uint16_t *>(rec + 8 * HS);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t w = c[4 * u] | c[4 * u + 1] << 4 | c[4 * u + 2] << 8 | c[4 * u + 3] << 12;
            codes[2 * word_of<HS>(half, 4 * (2 * t + u) + ((in & 7) >> 1), grp) + (in & 1)] = (uint16_t)w;
        }
    }
    if (t == 0) {
        reinterpret_cast<__half *>(rec + 16 * HS + (is_v ? HS : 0))[2 * ((in & 7) * groups(HS) + grp) + half] = scale;
        if ((__half_as_ushort(scale) & 0x7fffu) > KV4_ODD) a.kv.odd[slot] = 1u; // (whoever writes it writes the same)
    }
}

// ---- read-back: the values that the codes of some rows stand for -----------------------------------------------------------------------------------------------
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(bf16 *p, float v) { *p = __float2bfloat16_rn(v); }

template <int HS, typename T> __global__ void __launch_bounds__(256) k_read(View kv, Rows rows, T *__restrict__ k, T *__restrict__ v) {
    constexpr int L = HS / 8;
    pdl_wait();
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    const int li = (int)(item % L), G = kv.kv_heads, which = (int)(item / L % (2 * G));
    const long long row = item / L / (2 * G);
    if (row >= rows.n) return;
    const int pos = rows.position((int)row), slot = rows.slot_of((int)row);
    if (pos < 0 || pos >= kv.context || slot < 0 || slot >= kv.slots) return;
    const bool is_v = which >= G;
    const int head = is_v ? which - G : which, in = pos % BLOCK, half = in >> 3, grp = li >> 2, t = li & 3;
    const unsigned char *rec = record<HS>(kv, slot, head, pos / BLOCK);
    const float d = __half2float(reinterpret_cast<const __half *>(rec + 16 * HS + (is_v ? HS : 0))[2 * ((in & 7) * groups(HS) + grp) + half]);
    T *out = (is_v ? v : k) + (row * G + head) * HS + li * 8;
    int c[8];
    if (!is_v) {
        const uint32_t w = reinterpret_cast<const uint32_t *>(rec)[word_of<HS>(half, 4 * (in & 7) + t, grp)];
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = w >> (4 * (i >> 1) + 16 * (i & 1)) & 15;
    } else {
        const uint16_t *codes = reinterpret_cast<const uint16_t *>(rec + 8 * HS);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t w = codes[2 * word_of<HS>(half, 4 * (2 * t + u) + ((in & 7) >> 1), grp) + (in & 1)];
#pragma unroll
            for (int i = 0; i < 4; i++) c[4 * u + i] = w >> (4 * i) & 15;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) put(out + i, d * (float)(c[i] - 8));
}

// ---- attention of single rows ----------------------------------------------------------------------------------------------------------------------------------
struct Step {
    View kv;
    Rows rows;
    const float *q;
    long long ldq, ldo; // entries between rows
    int heads, window, vec, out_type;
    float scale;
    void *out;
    int8_t *quants; // out_type KV4_OUT_Q8: blocks of 32
    float *scales;
    float *work; // parts of units that several clusters share
    int by_length; // rows with the most positions first (at most STEP_ORDERED of them)
};

__device__ __forceinline__ float ex2(float x) { // 2^x
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { // d = a b
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// The codes of a word as pairs of FP16 numbers c - 8: pair i holds nibbles i and i + 4.  The bits of 1024 + c (or 1024 + 16 c) come from a mask, the rest is one exact operation.  (A masked
// code by itself is a number too, c 2^-24, but products of subnormals are added with as many bits less as they have leading zeros: 2^-17 in a score.)
__device__ __forceinline__ uint32_t magic() { // 1024 in both halves, in a register: a mask and an or with two literals would be two instructions
    uint32_t m;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m));
    return m;
}
__device__ __forceinline__ void unpack(uint32_t w, uint32_t one, uint32_t (&c)[4]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t v = i ? w >> 8 : w;
        uint32_t even, odd;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(even) : "r"(v), "n"(0x000f000f), "r"(one)); // (v & mask) | one
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(odd) : "r"(v), "n"(0x00f000f0), "r"(one));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(c[2 * i]) : "r"(even), "r"(0x64086408u));                                    // - 1032
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(c[2 * i + 1]) : "r"(odd), "r"(0x2c002c00u), "r"(0xd480d480u)); // / 16 - 72
    }
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp16_if(bool on, uint32_t dst, const void *src) { // predicated, not branched around
    asm volatile("{.reg .pred p; setp.ne.b32 p, %2, 0; @p cp.async.cg.shared.global [%0], [%1], 16;}" ::"r"(dst), "l"(src), "r"((int)on) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int VW> __device__ __forceinline__ void lds_words(const uint32_t *p, uint32_t (&w)[VW]) {
    if constexpr (VW == 4) { const uint4 v = *reinterpret_cast<const uint4 *>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (VW == 2) { const uint2 v = *reinterpret_cast<const uint2 *>(p); w[0] = v.x; w[1] = v.y; }
    else
#pragma unroll
        for (int i = 0; i < VW; i++) w[i] = p[i];
}

constexpr int STEP_WARPS = 8, STEP_MAX_CLUSTER = 8;
__host__ __device__ constexpr int step_records(int hs) { return hs >= 256 ? 1 : 2; }          // records that a warp takes at a time
__host__ __device__ constexpr int step_stages(int hs) { return hs >= 128 ? 3 : hs >= 64 ? 4 : 5; } // ... and has room for, with those under way
__host__ __device__ constexpr size_t step_ring_bytes(int hs) { return (size_t)STEP_WARPS * step_stages(hs) * step_records(hs) * record_bytes(hs); }
__host__ __device__ constexpr size_t step_merge_bytes(int hs, int heads) { return (size_t)(STEP_WARPS + 1) * heads * (hs + 2) * 4; } // the warps' parts and the CTA's
__host__ __device__ constexpr size_t step_smem_bytes(int hs, int heads) { return step_ring_bytes(hs) > step_merge_bytes(hs, heads) ? step_ring_bytes(hs) : step_merge_bytes(hs, heads); }

// The bounds of what row r sees: positions [lo, hi); none: lo >= hi.
__device__ __forceinline__ void visible(int pos, int window, int &lo, int &hi) {
    lo = window > 0 && pos >= window ? pos - window + 1 : 0;
    hi = pos + 1;
}
// One entry of a result row (whole warps, 32 neighbouring entries, where the blocks of 32 quants want them).
__device__ __forceinline__ void put_result(const Step &a, int row, size_t at, float v, bool on) {
    if (a.out_type == KV4_OUT_Q8) {
        float as;
        const int qv = quant_block_lane(v, as);
        if (on) {
            a.quants[row * a.ldo + at] = (int8_t)qv;
            if ((threadIdx.x & 31) == 0) a.scales[(row * a.ldo + at) / 32] = as;
        }
    } else if (!on) return;
    else if (a.out_type == B200_GGML_F32) ((float *)a.out)[row * a.ldo + at] = v;
    else if (a.out_type == B200_GGML_F16) put((__half *)a.out + row * a.ldo + at, v);
    else put((bf16 *)a.out + row * a.ldo + at, v);
}

// The row of a rank in the order of visible positions, most first and equal ones by index, so that the long rows of a batch do not start behind the short ones: a CTA ranks all rows, a row a
// thread.  us without / with it, 8 heads of 128 and of 64 up to 4096 positions: rows of any lengths 16: 26/23, 17/18, 24: 26/23, 19/15, 48: 43/35, 30/24; of one length (nothing to gain)
// 29/29, 19/19, 35/37, 21/21, 56/57, 35/35.  More rows cost more than they gain (96 rows of 2048 at most: 45/42, 27/25 and 60/65, 37/39; 200: 76/90, 45/60).
constexpr int STEP_ORDERED = 64;
__device__ __forceinline__ int row_by_length(const Step &a, int rank, int *lengths) { // lengths: 16-byte aligned, STEP_ORDERED + 1
    const int t = threadIdx.x;
    int length = -1;
    if (t < a.rows.n) {
        const int pos = a.rows.position(t), slot = a.rows.slot_of(t);
        int lo, hi;
        visible(pos, a.window, lo, hi);
        length = slot < 0 || slot >= a.kv.slots || pos >= a.kv.context || hi < lo ? 0 : hi - lo; // (padding: none)
    }
    if (t < STEP_ORDERED) lengths[t] = length;
    __syncthreads();
    if (t < a.rows.n) {
        int r = 0;
        for (int j = 0; j < a.rows.n; j += 4) {
            const int4 o = *reinterpret_cast<const int4 *>(lengths + j);
            r += (o.x > length || (o.x == length && j < t)) + (o.y > length || (o.y == length && j + 1 < t)) + (o.z > length || (o.z == length && j + 2 < t)) +
                 (o.w > length || (o.w == length && j + 3 < t));
        }
        if (r == rank) lengths[STEP_ORDERED] = t;
    }
    __syncthreads();
    const int row = __shfl_sync(0xffffffffu, lengths[STEP_ORDERED], 0);
    __syncthreads(); // (the memory is the ring's)
    return row;
}

// One query row and up to 4 NT query heads of a key/value head: the row's visible positions are split over the warps of a cluster of CTAs, each warp runs through its records
// (cp.async ring of its own, no barrier in the loop) with its own running maximum, and the parts are joined in shared memory, then over the cluster.  Where 8 CTAs a unit leave SMs
// idle, `splits` clusters share a unit: their parts go to the workspace, and k_step_join joins them.  Nothing depends on an order of arrival.
//   scores  C[16 positions x 8] = codes x queries in FP16; the eight columns are four heads, each as a high and a low part, so that a query keeps 22 bits; scaled group by group in FP32
//   values  C[16 entries x 8] = codes x (p d), again as a high and a low part.  p d is kept in FP16's range by a power of two that follows the largest value scale seen so far
// A lane keeps the running sums of ONE head (t); what crosses lanes in the loop is the transposition of the probabilities and, where a maximum grows by more than 2^8, its update.
// Bytes are its floor: 131071 positions of 8 heads of 128 are 151 MB, 23.4 us; it takes 36.5 (4.2 TB/s), 43.0 with the join and its gap.  What bounds it is how few warps an SM
// holds (two CTAs: 123 registers, 110 KB) and each one's chain: a record of 2304 bytes costs a warp about 300 instructions, half of them turning codes into FP16; a scheduler's four warps
// issue in 63 % of the cycles, with 1.5 of them ready, and wait for the arithmetic pipes (1.0 per issue), fixed latencies (0.65) and their records (0.56).  (The codes as they stand, subnormal FP16: fewer instructions, errors of 1e-5.)
template <int HS, int NT> __global__ void __launch_bounds__(STEP_WARPS * 32) k_step(const Step a, const int units_per_head, const int splits) {
    constexpr int NG = groups(HS), VW = vec_words(HS), R = record_bytes(HS), KB = step_records(HS), S = step_stages(HS), H = 4 * NT, CHUNKS = R / 16;
    extern __shared__ __align__(16) unsigned char smem[];
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.kv.kv_heads, mul = a.heads / G;
    const int split = blockIdx.x / ranks % splits, unit = blockIdx.x / ranks / splits, kvh = unit / units_per_head % G;
    const int first = unit % units_per_head * H; // first head within the group
    int row = unit / (G * units_per_head);
    if (a.by_length) row = row_by_length(a, row, reinterpret_cast<int *>(smem));
    const int pos = a.rows.position(row), slot = a.rows.slot_of(row);
    if (slot < 0 || slot >= a.kv.slots || pos >= a.kv.context) return; // a padding row (the whole cluster leaves)
    int lo, hi;
    visible(pos, a.window, lo, hi);
    const int workers = splits * ranks * STEP_WARPS, worker = (split * ranks + rank) * STEP_WARPS + warp;
    const int b0 = lo / BLOCK, nb = hi > lo ? (hi + BLOCK - 1) / BLOCK - b0 : 0, per = (nb + workers * KB - 1) / (workers * KB) * KB;
    const int begin = b0 + min(nb, worker * per), end = b0 + min(nb, (worker + 1) * per), stop = min(hi, end * BLOCK); // positions from `stop` on are none of this warp's

    unsigned char *ring = smem + (size_t)warp * S * KB * R;
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const unsigned char *src = record<HS>(a.kv, slot, kvh, begin) + lane * 16;
    int left = (end - begin) * CHUNKS - lane; // copies of 16 bytes, from this lane's first on
    auto fetch = [&](int stage) {
        const uint32_t d = ring_addr + stage * KB * R;
#pragma unroll
        for (int i = 0; i < (KB * CHUNKS + 31) / 32; i++) cp16_if(left > 32 * i && (32 * i + 31 < KB * CHUNKS || lane + 32 * i < KB * CHUNKS), d + i * 512, src + i * 512);
        src += KB * R;
        left -= KB * CHUNKS;
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; i++) fetch(i);

    // queries: lane (g, t) holds column g = head g >> 1, part g & 1, of entries 32 grp + 8 t .. + 7
    uint32_t qf[NT][NG][4];
    float sc[NT]; // of head t: what turns a sum into a score in units of log2
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int h = first + 4 * n + (g >> 1);
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int grp = 0; grp < NG; grp++) {
            if (h < mul) load8(a.q + row * a.ldq + (size_t)(kvh * mul + h) * HS + grp * 32 + t * 8, x[grp], a.vec);
            else
#pragma unroll
                for (int i = 0; i < 8; i++) x[grp][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[grp][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top) >> 23), 12), 230); // q times a power of two: below 1024, whatever its size
        const float up = __uint_as_float((unsigned)(263 - e) << 23), down = __uint_as_float((unsigned)(e - 9) << 23);
#pragma unroll
        for (int grp = 0; grp < NG; grp++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[grp][i] *= up;
                const float high = __half2float(__float2half_rn(x[grp][i]));
                x[grp][i] = g & 1 ? x[grp][i] - high : high;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) qf[n][grp][i] = pack_f16(x[grp][2 * i], x[grp][2 * i + 1]);
        }
        sc[n] = __shfl_sync(0xffffffffu, down, 8 * t) * (a.scale * 1.4426950408889634f);
    }

    float m[NT], l[NT], o[NT][2 * NG][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -CUDART_INF_F; l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NG; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }
    int lift = 0;            // p d is held times 2^lift
    uint32_t most = 0u;      // scales up to here (their bits) have been seen: 2^lift * scale < 2^7
    const uint32_t one = magic();
    int stage = 0;
#pragma unroll 1
    for (int block = begin; block < end; block += KB) {
        cp_wait<S - 2>();
        __syncwarp(); // and every lane has read the stage that the next copy overwrites
        fetch(stage == 0 ? S - 1 : stage - 1);
        const uint32_t *words = reinterpret_cast<const uint32_t *>(ring + stage * KB * R);
        float s[KB][NT][2];
        uint32_t dv[KB][NG]; // value scales of positions g and g + 8
#pragma unroll
        for (int b = 0; b < KB; b++) {
            const uint32_t *codes = words + b * (R / 4), *ks = codes + 4 * HS + g * NG;
#pragma unroll
            for (int n = 0; n < NT; n++) s[b][n][0] = s[b][n][1] = 0.0f;
#pragma unroll
            for (int v = 0; v < NG / VW; v++) {
                uint32_t wa[VW], wb[VW], d[VW], dw[VW];
                lds_words<VW>(codes + word_of<HS>(0, lane, v * VW), wa);
                lds_words<VW>(codes + word_of<HS>(1, lane, v * VW), wb);
                lds_words<VW>(ks + v * VW, d);
                lds_words<VW>(ks + 8 * NG + v * VW, dw);
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    const int grp = v * VW + i;
                    dv[b][grp] = dw[i];
                    uint32_t ca[4], cb[4];
                    unpack(wa[i], one, ca);
                    unpack(wb[i], one, cb);
                    const uint32_t c0[4] = {ca[0], cb[0], ca[1], cb[1]}, c1[4] = {ca[2], cb[2], ca[3], cb[3]};
                    const float2 dk = __half22float2(*reinterpret_cast<const __half2 *>(&d[i]));
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float acc[4];
                        mma_f16_first(acc, c0, qf[n][grp][0], qf[n][grp][1]);
                        mma_f16(acc, c1, qf[n][grp][2], qf[n][grp][3]);
                        s[b][n][0] = fmaf(dk.x, acc[0] + acc[1], s[b][n][0]);
                        s[b][n][1] = fmaf(dk.y, acc[2] + acc[3], s[b][n][1]);
                    }
                }
            }
        }
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int n = 0; n < NT; n++) { s[b][n][0] *= sc[n]; s[b][n][1] *= sc[n]; }
        if (block * BLOCK < lo || (block + KB) * BLOCK > stop) { // an end of what the warp takes: whatever stands behind it has no weight and no scale
#pragma unroll
            for (int b = 0; b < KB; b++) {
                const int p0 = (block + b) * BLOCK + g;
                const bool see0 = p0 >= lo && p0 < stop, see1 = p0 + 8 >= lo && p0 + 8 < stop;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if (!see0) s[b][n][0] = -CUDART_INF_F;
                    if (!see1) s[b][n][1] = -CUDART_INF_F;
                }
#pragma unroll
                for (int grp = 0; grp < NG; grp++) dv[b][grp] &= (see0 ? 0xffffu : 0u) | (see1 ? 0xffff0000u : 0u);
            }
        }
        __half2 widest = __habs2(*reinterpret_cast<const __half2 *>(&dv[0][0])); // (NaN loses against a number)
#pragma unroll
        for (int grp = 1; grp < KB * NG; grp++) widest = __hmax2(widest, __habs2(*reinterpret_cast<const __half2 *>(&dv[grp / NG][grp % NG])));
        const uint32_t wide = *reinterpret_cast<const uint32_t *>(&widest);
        bool rare = ((0x80008000u + most * 0x10001u) - wide & 0x80008000u) != 0x80008000u; // a half of it above `most`
        float mx[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            mx[n] = fmaxf(s[0][n][0], s[0][n][1]);
#pragma unroll
            for (int b = 1; b < KB; b++) mx[n] = fmaxf(mx[n], fmaxf(s[b][n][0], s[b][n][1]));
            rare |= mx[n] > m[n] + 8.0f;
        }
        if (__any_sync(0xffffffffu, rare)) {
            const uint32_t big = __reduce_max_sync(0xffffffffu, max(wide & 0xffffu, wide >> 16));
            float beta = 1.0f;
            if (big > most && big <= 0x7c00u) { // (a NaN changes nothing)
                const int was = lift;
                lift = 21 - (int)(big >> 10); // the scale is below 2^(big >> 10 - 14)
                if (most) beta = __uint_as_float((unsigned)(127 + lift - was) << 23); // (no sums before the first scale)
                most = big | 0x3ffu;
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], i));
                mx[n] = fmaxf(mx[n], m[n]);
                const float alpha = m[n] == mx[n] ? 1.0f : ex2(m[n] - mx[n]), gamma = alpha * beta;
                m[n] = mx[n];
                l[n] *= alpha;
#pragma unroll
                for (int i = 0; i < 2 * NG; i++) { o[n][i][0] *= gamma; o[n][i][1] *= gamma; o[n][i][2] *= gamma; o[n][i][3] *= gamma; }
            }
        }
        const float two_to_lift = __uint_as_float((unsigned)(127 + lift) << 23);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float ref = m[n] == -CUDART_INF_F ? 0.0f : m[n]; // nothing seen yet: 2^(-inf) = 0
#pragma unroll
            for (int b = 0; b < KB; b++) {
                s[b][n][0] = ex2(s[b][n][0] - ref);
                s[b][n][1] = ex2(s[b][n][1] - ref);
                l[n] += s[b][n][0] + s[b][n][1];
                s[b][n][0] *= two_to_lift;
                s[b][n][1] *= two_to_lift;
            }
        }
#pragma unroll
        for (int b = 0; b < KB; b++) {
            const uint32_t *codes = words + b * (R / 4) + 2 * HS;
#pragma unroll
            for (int v = 0; v < NG / VW; v++) {
                uint32_t wa[VW], wb[VW];
                lds_words<VW>(codes + word_of<HS>(0, lane, v * VW), wa);
                lds_words<VW>(codes + word_of<HS>(1, lane, v * VW), wb);
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    const int grp = v * VW + i;
                    const float2 d = __half22float2(*reinterpret_cast<const __half2 *>(&dv[b][grp]));
                    uint32_t ca[4], cb[4];
                    unpack(wa[i], one, ca);
                    unpack(wb[i], one, cb);
                    const uint32_t c0[4] = {ca[0], ca[1], cb[0], cb[1]}, c1[4] = {ca[2], ca[3], cb[2], cb[3]};
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float x0 = s[b][n][0] * d.x, x1 = s[b][n][1] * d.y; // the high part: the 11 bits that FP16 has, cut off
                        const float h0 = __uint_as_float(__float_as_uint(x0) & 0xffffe000u), h1 = __uint_as_float(__float_as_uint(x1) & 0xffffe000u);
                        const uint32_t f0 = transpose8x8(pack_f16(h0, x0 - h0)), f1 = transpose8x8(pack_f16(h1, x1 - h1));
                        mma_f16(o[n][2 * grp], c0, f0, f1);
                        mma_f16(o[n][2 * grp + 1], c1, f0, f1);
                    }
                }
            }
        }
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncthreads();

    // ---- join: warps, then CTAs, then (through the workspace) clusters -------------------------------------------------------------------------------------------
    float *part = reinterpret_cast<float *>(smem), *pm = part + (STEP_WARPS + 1) * H * HS, *pl = pm + (STEP_WARPS + 1) * H; // [warp, or the CTA's][head][entry]
    const float unit_of = __uint_as_float((unsigned)(127 - lift) << 23);
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], i);
        const int h = 4 * n + t;
        if (g == 0) { pm[warp * H + h] = m[n]; pl[warp * H + h] = l[n]; }
#pragma unroll
        for (int grp = 0; grp < NG; grp++)
            *reinterpret_cast<float4 *>(part + (warp * H + h) * HS + grp * 32 + g * 4) =
                make_float4((o[n][2 * grp][0] + o[n][2 * grp][1]) * unit_of, (o[n][2 * grp][2] + o[n][2 * grp][3]) * unit_of, (o[n][2 * grp + 1][0] + o[n][2 * grp + 1][1]) * unit_of,
                            (o[n][2 * grp + 1][2] + o[n][2 * grp + 1][3]) * unit_of);
    }
    __syncthreads();
    const int mine = STEP_WARPS * H; // rows behind the warps': the CTA's
    for (int i = threadIdx.x; i < H * HS; i += STEP_WARPS * 32) {
        const int h = i / HS;
        float M = -CUDART_INF_F, L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) M = fmaxf(M, pm[w * H + h]);
        const float ref = M == -CUDART_INF_F ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; w++) {
            const float f = ex2(pm[w * H + h] - ref);
            L = fmaf(f, pl[w * H + h], L);
            O = fmaf(f, part[(w * H) * HS + i], O);
        }
        part[mine * HS + i] = O;
        if (i % HS == 0) { pm[mine + h] = M; pl[mine + h] = L; }
    }
    if (ranks > 1) cluster.sync(); else __syncthreads();
    const int slice = H * HS / ranks;
    for (int j = threadIdx.x; j < slice; j += STEP_WARPS * 32) { // (whole warps: slice is a multiple of 32 where blocks of 32 quants need it)
        const int i = rank * slice + j, h = i / HS;
        float M = -CUDART_INF_F, L = 0.0f, O = 0.0f;
        for (int r = 0; r < ranks; r++) M = fmaxf(M, *cluster.map_shared_rank(pm + mine + h, r));
        const float ref = M == -CUDART_INF_F ? 0.0f : M;
        for (int r = 0; r < ranks; r++) {
            const float f = ex2(*cluster.map_shared_rank(pm + mine + h, r) - ref);
            L = fmaf(f, *cluster.map_shared_rank(pl + mine + h, r), L);
            O = fmaf(f, *cluster.map_shared_rank(part + mine * HS + i, r), O);
        }
        if (splits > 1) { // [row][head][split]: maximum, sum, entries
            if (first + h < mul) {
                float *w = a.work + (((size_t)row * a.heads + kvh * mul + first + h) * splits + split) * (HS + 2);
                w[2 + i % HS] = O;
                if (i % HS == 0) { w[0] = M; w[1] = L; }
            }
        } else put_result(a, row, (size_t)(kvh * mul + first + h) * HS + i % HS, hi <= lo ? 0.0f : O / L, first + h < mul); // a row that sees nothing: zeros
    }
    if (ranks > 1) cluster.sync(); // no CTA leaves while another reads its part
}

// Joins the parts of a row's head: the weights of the splits once, then an entry a thread.  At most STEP_MAX_SPLITS parts.
constexpr int STEP_MAX_SPLITS = 296;
template <int HS> __global__ void __launch_bounds__(HS < 64 ? 64 : HS) k_step_join(const Step a, const int splits) {
    constexpr int HEADS = HS < 64 ? 64 / HS : 1, LD = HS + 2; // heads of a CTA
    __shared__ float weight[HEADS][STEP_MAX_SPLITS], sum[HEADS][STEP_MAX_SPLITS];
    pdl_wait();
    const int at = threadIdx.x / HS, h = blockIdx.x % ((a.heads + HEADS - 1) / HEADS) * HEADS + at, row = blockIdx.x / ((a.heads + HEADS - 1) / HEADS), i = threadIdx.x % HS;
    const int pos = a.rows.position(row), slot = a.rows.slot_of(row);
    if (slot < 0 || slot >= a.kv.slots || pos >= a.kv.context) return;
    const bool on = h < a.heads;
    int lo, hi;
    visible(pos, a.window, lo, hi);
    const float *w = a.work + ((size_t)row * a.heads + (on ? h : 0)) * splits * LD;
    for (int s = i; s < splits; s += HS) { weight[at][s] = w[s * LD]; sum[at][s] = w[s * LD + 1]; }
    __syncthreads();
    float M = -CUDART_INF_F, L = 0.0f, O = 0.0f;
    for (int s = 0; s < splits; s++) M = fmaxf(M, weight[at][s]);
    const float ref = M == -CUDART_INF_F ? 0.0f : M;
    __syncthreads();
    for (int s = i; s < splits; s += HS) weight[at][s] = ex2(weight[at][s] - ref);
    __syncthreads();
#pragma unroll 8
    for (int s = 0; s < splits; s++) {
        L = fmaf(weight[at][s], sum[at][s], L);
        O = fmaf(weight[at][s], w[s * LD + 2 + i], O);
    }
    put_result(a, row, (size_t)h * HS + i, hi <= lo ? 0.0f : O / L, on);
}

} // namespace kv4
