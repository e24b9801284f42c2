// operators.cu -- libb200llama.so: operators that work on a caller's device memory and stream (b200_kv4_*, b200_log_probs) and that plans call on theirs.
#include "operators.h"
#include "kv4_chunk.cuh"
#include "logprobs.cuh"
#include "operator_util.cuh"

#include <stdlib.h>
#include <string.h>

#include <new>

struct b200_kv4 {
    kv4::View view{};
    int head_size = 0, device = 0, sms = 148;
    size_t bytes = 0;
    unsigned *host_error = nullptr, *device_error = nullptr; // a mapped word: what a wait that gave up leaves (kv4_chunk.cuh)
    char err[256] = "";
    size_t marks_bytes() const { return (size_t)view.slots * 4; } // behind the records: View::odd, and a word that no reset clears
};

namespace {

template <typename... A> int fail(b200_kv4 *kv, int code, const char *fmt, A... a) { return say(kv->err, sizeof kv->err, code, fmt, a...); }
bool refused(const char *step) { // (as in plan.cu: what tests refuse)
    const char *e = getenv("B200_TEST_REFUSE");
    return e && strstr(e, step);
}

} // namespace

cudaError_t kv4_append_launch(const b200_kv4 *kv, const b200_kv4_append_args &a, cudaStream_t stream, bool pdl) {
    kv4::Append k;
    k.kv = kv->view;
    k.rows = {a.positions, a.slots, a.n, a.start, a.slot};
    k.q = a.q; k.k = a.k; k.v = a.v;
    k.ldq = a.q_stride; k.ldk = a.k_stride; k.ldv = a.v_stride; k.ldo = a.q_out_stride;
    k.heads = a.heads;
    k.interleaved = a.rope_layout == B200_ROPE_INTERLEAVED;
    const int b = type_bytes(a.type);
    k.vec = aligned16(a.k, a.k_stride, b) && aligned16(a.v, a.v_stride, b) && (!a.heads || (aligned16(a.q, a.q_stride, b) && aligned16(a.q_out, a.q_out_stride, 4)));
    k.q_norm = a.q_norm; k.k_norm = a.k_norm; k.cos = a.cos; k.sin = a.sin;
    k.eps = a.eps;
    k.q_out = a.q_out;
    return by_head_size(kv->head_size, [&](auto hs) {
        return by_type(a.type, [&](auto type) {
            constexpr int L = hs / 8, per_warp = L == 4 ? 8 : L == 8 ? 4 : L <= 16 ? 2 : 1;
            const long long items = (long long)a.n * (a.heads + 2 * kv->view.kv_heads);
            return launch(kv4::k_append<hs, decltype(type)>, (unsigned)((items + 8 * per_warp - 1) / (8 * per_warp)), 256, 0, 1, pdl, stream, k);
        });
    });
}

// How the work of single rows is cut: heads of a unit, units of a row and key/value head, CTAs of a cluster, clusters of a unit.
struct StepCut {
    int heads, per_head, cluster, splits;
};
static StepCut step_cut(const b200_kv4 *kv, const b200_kv4_attention_args &a, bool quants) {
    StepCut c;
    const int G = kv->view.kv_heads, mul = a.heads / G, hs = kv->head_size;
    c.heads = mul > 4 && hs < 256 ? 8 : 4;
    c.per_head = (mul + c.heads - 1) / c.heads;
    const long long units = (long long)a.n * G * c.per_head;
    const int len = a.max_len > 0 && a.max_len < kv->view.context ? a.max_len : kv->view.context, seen = a.window > 0 && a.window < len ? a.window : len;
    const int group = kv4::BLOCK * kv4::step_records(hs) * kv4::STEP_WARPS; // positions that a CTA takes at a time
    // Few units over many positions: two CTAs for every SM, evenly, through the workspace (clusters of 8 leave SMs with one CTA beside SMs with two: the kernel took 42 us for 131071
    // positions of 8 heads, cut evenly 36.6).
    c.splits = units * kv4::STEP_MAX_CLUSTER < 2 * kv->sms && seen >= 4 * group * kv4::STEP_MAX_CLUSTER ? (int)(2 * kv->sms / units) : 1;
    if (c.splits > seen / (4 * group)) c.splits = seen / (4 * group); // at least four rounds a warp
    if (c.splits < 1) c.splits = 1;
    if (c.splits > kv4::STEP_MAX_SPLITS) c.splits = kv4::STEP_MAX_SPLITS;
    int most = (seen + group - 1) / group;
    if (most > kv4::STEP_MAX_CLUSTER) most = kv4::STEP_MAX_CLUSTER;
    c.cluster = cluster_for(units, 4 * kv->sms, most); // (more CTAs cost more in front and behind than they spread: 16 rows of 8 heads of 128 over 4096 positions 29 us, with twice as many 39)
    // whole blocks of 32 quants a CTA: heads of 96 in units of four are 12 blocks, of which 8 CTAs would have one and a half each
    while (quants && c.heads * hs / c.cluster % 32) c.cluster /= 2;
    return c;
}
static size_t parts_bytes(const b200_kv4 *kv, const b200_kv4_attention_args &a, int splits) { return splits > 1 ? (size_t)a.n * a.heads * splits * (kv->head_size + 2) * 4 : 0; }

// Chunks on the tensor cores: 16-bit results, heads of 64, 96 or 128.  A tile takes 128 rows whether they are used or not, single rows read the cache once each.  us as single rows / as a chunk,
// by rows (tokens x query heads of a key/value head):  32/8 heads of 128, 8192 positions: 32 rows 29/25, 64 rows 53/25, 128 rows 76/27;  1024 positions: 11/21, 17/21, 29/23;
// 32/8 heads of 64, 8192: 21/23, 33/23, 47/23;  16/16 of 64, 4096: 41/23 (32 rows), 66/23;  8/1 of 128, 8192: 17/25, 17/25, 17/27, 60/27 (512 rows).
// The rule looks at a key/value head's rows alone: 64 of them over 1024 positions, and 64 to 128 of a single head, take the slower form, by 4 to 10 us.
const int CHUNK_MIN_ROWS = 64;
struct ChunkCut {
    int tokens, splits;
    bool use;
};
static ChunkCut chunk_cut(const b200_kv4 *kv, const b200_kv4_attention_args &a, bool quants) {
    ChunkCut c = {};
    const int G = kv->view.kv_heads, mul = a.heads / G, hs = kv->head_size;
    const int chunk = a.chunk < a.n ? a.chunk : a.n;
    c.use = !quants && a.out_type != B200_GGML_F32 && (hs == 64 || hs == 96 || hs == 128) && mul <= kv4::CHUNK_ROWS && chunk > 1 && (long long)chunk * mul >= CHUNK_MIN_ROWS;
    if (!c.use) return c;
    const int len = a.max_len > 0 && a.max_len < kv->view.context ? a.max_len : kv->view.context;
    // even shares of a chunk, so that where all rows are chunks of that many tokens no CTA has two sequences' positions to run through (three chunks of 111, 42 tokens at most: 21 us, not 31)
    const int most = kv4::CHUNK_ROWS / mul, shares = (chunk + most - 1) / most;
    c.tokens = (chunk + shares - 1) / shares;
    const long long units = (long long)((a.n + c.tokens - 1) / c.tokens) * G;
    const long long near = (long long)a.window + c.tokens, seen = a.window > 0 && near < len ? near : len, worth = seen / (8 * kv4::CHUNK_KEYS); // eight tiles of positions a CTA
    long long splits = kv->sms / units;
    if (splits > worth) splits = worth;
    c.splits = splits < 1 ? 1 : (int)splits;
    return c;
}

static cudaError_t attention_launch(const b200_kv4 *kv, const b200_kv4_attention_args &a, int8_t *quants, float *scales, cudaStream_t stream, bool pdl, int *launches, bool give_up) {
    kv4::Step k;
    k.kv = kv->view;
    k.rows = {a.positions, a.slots, a.n, a.start, a.slot};
    k.q = a.q;
    k.ldq = a.q_stride; k.ldo = a.out_stride;
    k.heads = a.heads; k.window = a.window;
    k.vec = aligned16(a.q, a.q_stride, 4);
    k.out_type = quants ? KV4_OUT_Q8 : a.out_type;
    k.scale = a.scale;
    k.out = a.out; k.quants = quants; k.scales = scales;
    k.work = a.workspace;
    k.by_length = 0;
    const auto has_room = [&](int splits) { return a.workspace && parts_bytes(kv, a, splits) <= a.workspace_bytes; };
    const auto join = [&](auto hs, int splits) {
        constexpr int per_cta = hs < 64 ? 64 / hs : 1;
        return launch(kv4::k_step_join<hs>, (unsigned)a.n * ((a.heads + per_cta - 1) / per_cta), hs < 64 ? 64 : hs, 0, 1, true, stream, k, splits);
    };
    ChunkCut cc = chunk_cut(kv, a, quants != nullptr);
    if (cc.use) {
        if (!has_room(cc.splits)) cc.splits = 1;
        if (launches) *launches = cc.splits > 1 ? 2 : 1;
        kv4::Chunk ck = {k, cc.tokens, cc.splits, aligned16(a.out, a.out_stride, 2), kv->device_error};
        const unsigned grid = (unsigned)((a.n + cc.tokens - 1) / cc.tokens) * kv->view.kv_heads * cc.splits;
        const auto go = [&](auto hs) {
            constexpr size_t smem = kv4::chunk_smem_bytes(hs);
            auto kern = kv4::k_chunk<hs>;
            if constexpr (hs == 64) if (give_up) kern = kv4::k_chunk<hs, true>;
            cudaError_t e = allow_smem(kern, smem);
            if (e == cudaSuccess) e = launch(kern, grid, kv4::CHUNK_THREADS, smem, 1, pdl, stream, ck);
            return e != cudaSuccess || cc.splits == 1 ? e : join(hs, cc.splits);
        };
        if (kv->head_size == 64) return go(std::integral_constant<int, 64>());
        if (kv->head_size == 96) return go(std::integral_constant<int, 96>());
        return go(std::integral_constant<int, 128>());
    }
    StepCut c = step_cut(kv, a, quants != nullptr);
    if (c.splits > 1 && has_room(c.splits)) c.cluster = 1;
    else c.splits = 1;
    if (launches) *launches = c.splits > 1 ? 2 : 1;
    return by_head_size(kv->head_size, [&](auto hs) {
        auto go = [&](auto nt) {
            constexpr size_t smem = kv4::step_smem_bytes(hs, 4 * nt);
            const unsigned grid = (unsigned)a.n * kv->view.kv_heads * c.per_head * c.splits * c.cluster;
            k.by_length = a.positions && a.n > 1 && a.n <= kv4::STEP_ORDERED && grid > 2u * kv->sms;
            auto kern = kv4::k_step<hs, nt>;
            cudaError_t e = allow_smem(kern, smem);
            if (e == cudaSuccess) e = launch(kern, grid, kv4::STEP_WARPS * 32, smem, c.cluster, pdl, stream, k, c.per_head, c.splits);
            return e != cudaSuccess || c.splits == 1 ? e : join(hs, c.splits);
        };
        if constexpr (hs < 256) if (c.heads == 8) return go(std::integral_constant<int, 2>());
        return go(std::integral_constant<int, 1>());
    });
}

cudaError_t kv4_attention_launch(const b200_kv4 *kv, const b200_kv4_attention_args &a, int8_t *quants, float *scales, cudaStream_t stream, bool pdl, int *launches) {
    return attention_launch(kv, a, quants, scales, stream, pdl, launches, false);
}

bool kv4_gave_up(const b200_kv4 *kv) { return *reinterpret_cast<volatile unsigned *>(kv->host_error); }

cudaError_t log_probs_launch(const b200_log_probs_args &a, cudaStream_t stream) {
    lp::Args k;
    k.logits = a.logits;
    k.ld = a.row_stride;
    k.rows = a.rows; k.vocab = a.vocab; k.top = a.top;
    k.targets = a.targets;
    k.logprobs = a.logprobs; k.entropy = a.entropy; k.top_logprobs = a.top_logprobs;
    k.top_ids = a.top_ids;
    const long long most = (a.vocab + 2047) / 2048;
    const int cluster = cluster_for(a.rows, 4LL * sm_count(a.device), most < lp::MAX_CLUSTER ? most : lp::MAX_CLUSTER);
    return by_type(a.type, [&](auto type) {
        return launch(lp::k_log_probs<decltype(type)>, (unsigned)a.rows * cluster, lp::THREADS, 0, cluster, false, stream, k);
    });
}

extern "C" {

int b200_kv4_create(int32_t slots, int32_t context, int32_t kv_heads, int32_t head_size, int32_t device, b200_kv4 **out, char *err, size_t err_len) {
    if (out) *out = nullptr;
    if (!out) return say(err, err_len, B200_ERR_BAD_ARG, "null argument");
    if (slots <= 0 || context <= 0 || kv_heads <= 0 || context > INT32_MAX - 64) return say(err, err_len, B200_ERR_BAD_ARG, "slots, context and kv_heads must be positive");
    if (head_size != 32 && head_size != 64 && head_size != 96 && head_size != 128 && head_size != 256)
        return say(err, err_len, B200_ERR_UNSUPPORTED, "a 4-bit cache has heads of 32, 64, 96, 128 or 256 entries, not %d", head_size);
    int devices = 0;
    cudaError_t e = cudaGetDeviceCount(&devices);
    if (e != cudaSuccess) return say(err, err_len, B200_ERR_CUDA, "%s", cudaGetErrorString(e));
    if (device < 0 || device >= devices) return say(err, err_len, B200_ERR_BAD_ARG, "device %d of %d", device, devices);
    b200_kv4 *kv = new (std::nothrow) b200_kv4();
    if (!kv) return say(err, err_len, B200_ERR_OOM, "no host memory");
    kv->head_size = head_size;
    kv->device = device;
    kv->sms = sm_count(device);
    kv->view = {nullptr, nullptr, slots, context, (context + kv4::BLOCK - 1) / kv4::BLOCK, kv_heads};
    const unsigned __int128 bytes = (unsigned __int128)slots * kv_heads * kv->view.blocks * kv4::record_bytes(head_size);
    OnDevice on(device);
    e = on.error;
    if (e == cudaSuccess) e = bytes > ((unsigned __int128)1 << 48) ? cudaErrorMemoryAllocation : cudaMalloc((void **)&kv->view.base, (size_t)bytes + kv->marks_bytes() + 4);
    if (e == cudaSuccess) {
        kv->bytes = (size_t)bytes;
        kv->view.odd = reinterpret_cast<unsigned *>(kv->view.base + kv->bytes); // (records are multiples of 64 bytes)
        e = cudaMemset(kv->view.base, 0, kv->bytes + kv->marks_bytes() + 4);
        if (e == cudaSuccess) e = cudaDeviceSynchronize(); // the memory is zeros for every stream
    }
    // the word through which a wait that gave up is heard of: no cache without it
    if (e == cudaSuccess) e = refused("kv4_word") ? cudaErrorMemoryAllocation : cudaHostAlloc((void **)&kv->host_error, 4, cudaHostAllocMapped);
    if (e == cudaSuccess) {
        *kv->host_error = 0;
        e = cudaHostGetDevicePointer((void **)&kv->device_error, kv->host_error, 0);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        say(err, err_len, 0, "4-bit cache of %.3g GB: %s", (double)bytes / 1e9, cudaGetErrorString(e));
        cudaFree(kv->view.base);
        cudaFreeHost(kv->host_error);
        delete kv;
        return cuda_code(e);
    }
    *out = kv;
    return B200_OK;
}

void b200_kv4_free(b200_kv4 *kv) {
    if (!kv) return;
    OnDevice on(kv->device);
    cudaFree(kv->view.base); // (waits for the device's work)
    cudaFreeHost(kv->host_error);
    delete kv;
}

int64_t b200_kv4_device_bytes(const b200_kv4 *kv) { return kv ? (int64_t)kv->bytes : 0; }
const char *b200_kv4_last_error(const b200_kv4 *kv) { return kv ? kv->err : "null cache"; }

int b200_kv4_reset(b200_kv4 *kv, void *stream) {
    if (!kv) return B200_ERR_BAD_ARG;
    OnDevice on(kv->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->view.base, 0, kv->bytes + kv->marks_bytes(), (cudaStream_t)stream);
    return e == cudaSuccess ? B200_OK : fail(kv, cuda_code(e), "%s", cudaGetErrorString(e));
}

static int check_error(b200_kv4 *kv) {
    if (kv4_gave_up(kv))
        return fail(kv, B200_ERR_STATE, "an earlier attention of a chunk gave up a wait on the device: its results, and what came of them, are not valid; the cache must be freed");
    return B200_OK;
}

static int check_rows(b200_kv4 *kv, int n, const int32_t *positions, int32_t start, const int32_t *slots, int32_t slot) {
    if (n < 0) return fail(kv, B200_ERR_BAD_ARG, "%d rows", n);
    if (!slots && (slot < 0 || slot >= kv->view.slots)) return fail(kv, B200_ERR_BAD_ARG, "slot %d of %d", slot, kv->view.slots);
    if (!positions && (start < 0 || (long long)start + n > kv->view.context)) return fail(kv, B200_ERR_BAD_ARG, "positions %d .. %lld outside the cache (%d)", start, (long long)start + n - 1, kv->view.context);
    return B200_OK;
}

int b200_kv4_append(b200_kv4 *kv, const b200_kv4_append_args *a, void *stream) {
    if (!kv) return B200_ERR_BAD_ARG;
    if (!a) return fail(kv, B200_ERR_BAD_ARG, "null arguments");
    int rc = check_rows(kv, a->n, a->positions, a->start, a->slots, a->slot);
    if (rc) return rc;
    if (a->heads < 0) return fail(kv, B200_ERR_BAD_ARG, "%d query heads", a->heads);
    if (!known_type(a->type)) return fail(kv, B200_ERR_UNSUPPORTED, "rows of type %d (FP32, FP16 and BF16 are known)", a->type);
    if (a->rope_layout != B200_ROPE_HALF && a->rope_layout != B200_ROPE_INTERLEAVED) return fail(kv, B200_ERR_BAD_ARG, "rotation layout %d", a->rope_layout);
    if (!a->cos != !a->sin) return fail(kv, B200_ERR_BAD_ARG, "a rotation needs both tables");
    if (a->n == 0) return B200_OK;
    if (!a->k || !a->v || (a->heads && (!a->q || !a->q_out))) return fail(kv, B200_ERR_BAD_ARG, "null rows");
    const int64_t kv_width = (int64_t)kv->view.kv_heads * kv->head_size, q_width = (int64_t)a->heads * kv->head_size;
    if (a->k_stride < kv_width || a->v_stride < kv_width || (a->heads && (a->q_stride < q_width || a->q_out_stride < q_width))) return fail(kv, B200_ERR_BAD_ARG, "rows overlap: a stride is smaller than its row");
    if ((long long)a->n * (a->heads + 2 * kv->view.kv_heads) > (1LL << 33)) return fail(kv, B200_ERR_UNSUPPORTED, "too many rows in one call");
    OnDevice on(kv->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess) e = kv4_append_launch(kv, *a, (cudaStream_t)stream, false);
    return e == cudaSuccess ? B200_OK : fail(kv, cuda_code(e), "%s", cudaGetErrorString(e));
}

static int attention(b200_kv4 *kv, const b200_kv4_attention_args *a, void *stream, bool give_up) {
    if (!kv) return B200_ERR_BAD_ARG;
    if (!a) return fail(kv, B200_ERR_BAD_ARG, "null arguments");
    int rc = check_error(kv);
    if (!rc) rc = check_rows(kv, a->n, a->positions, a->start, a->slots, a->slot);
    if (rc) return rc;
    if (a->heads <= 0 || a->heads % kv->view.kv_heads) return fail(kv, B200_ERR_BAD_ARG, "%d query heads over %d key/value heads", a->heads, kv->view.kv_heads);
    if (!known_type(a->out_type)) return fail(kv, B200_ERR_UNSUPPORTED, "results of type %d (FP32, FP16 and BF16 are known)", a->out_type);
    if (reinterpret_cast<uintptr_t>(a->workspace) % 16) return fail(kv, B200_ERR_BAD_ARG, "the workspace is not aligned");
    if (a->window < 0 || a->max_len < 0 || a->chunk < 0) return fail(kv, B200_ERR_BAD_ARG, "a negative window, length or chunk");
    if (a->n == 0) return B200_OK;
    if (!a->q || !a->out) return fail(kv, B200_ERR_BAD_ARG, "null rows");
    const int64_t width = (int64_t)a->heads * kv->head_size;
    if (a->q_stride < width || a->out_stride < width) return fail(kv, B200_ERR_BAD_ARG, "rows overlap: a stride is smaller than its row");
    if ((long long)a->n * a->heads > (1LL << 27)) return fail(kv, B200_ERR_UNSUPPORTED, "too many rows in one call");
    OnDevice on(kv->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess) e = attention_launch(kv, *a, nullptr, nullptr, (cudaStream_t)stream, false, nullptr, give_up);
    return e == cudaSuccess ? B200_OK : fail(kv, cuda_code(e), "%s", cudaGetErrorString(e));
}
int b200_kv4_attention(b200_kv4 *kv, const b200_kv4_attention_args *a, void *stream) { return attention(kv, a, stream, false); }
int b200_test_kv4_give_up(b200_kv4 *kv, const b200_kv4_attention_args *a, void *stream) {
    if (!kv) return B200_ERR_BAD_ARG;
    if (!a || a->n <= 0 || a->heads <= 0 || a->heads % kv->view.kv_heads || kv->head_size != 64 || !chunk_cut(kv, *a, false).use)
        return fail(kv, B200_ERR_BAD_ARG, "no attention of a chunk with heads of 64");
    return attention(kv, a, stream, true);
}

size_t b200_kv4_attention_workspace(const b200_kv4 *kv, const b200_kv4_attention_args *a) {
    if (!kv || !a || a->n <= 0 || a->heads <= 0 || a->heads % kv->view.kv_heads) return 0;
    const ChunkCut c = chunk_cut(kv, *a, false);
    return parts_bytes(kv, *a, c.use ? c.splits : step_cut(kv, *a, false).splits);
}

int b200_kv4_read(b200_kv4 *kv, const b200_kv4_read_args *a, void *stream) {
    if (!kv) return B200_ERR_BAD_ARG;
    if (!a) return fail(kv, B200_ERR_BAD_ARG, "null arguments");
    int rc = check_rows(kv, a->n, a->positions, a->start, a->slots, a->slot);
    if (rc) return rc;
    if (!known_type(a->type)) return fail(kv, B200_ERR_UNSUPPORTED, "rows of type %d (FP32, FP16 and BF16 are known)", a->type);
    if (a->n == 0) return B200_OK;
    if (!a->k || !a->v) return fail(kv, B200_ERR_BAD_ARG, "null rows");
    if ((long long)a->n * kv->view.kv_heads > (1LL << 33)) return fail(kv, B200_ERR_UNSUPPORTED, "too many rows in one call");
    OnDevice on(kv->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess)
        e = by_head_size(kv->head_size, [&](auto hs) {
            return by_type(a->type, [&](auto type) {
                using T = decltype(type);
                const long long items = (long long)a->n * 2 * kv->view.kv_heads * (hs / 8);
                const kv4::Rows rows = {a->positions, a->slots, a->n, a->start, a->slot};
                return launch(kv4::k_read<hs, T>, (unsigned)((items + 255) / 256), 256, 0, 1, false, (cudaStream_t)stream, kv->view, rows, (T *)a->k, (T *)a->v);
            });
        });
    return e == cudaSuccess ? B200_OK : fail(kv, cuda_code(e), "%s", cudaGetErrorString(e));
}

int b200_test_kv4_step_cut(int32_t head_size, int32_t kv_heads, int32_t heads, int32_t n, int32_t context, int32_t max_len, int32_t window, int32_t sms, int32_t quants, int32_t *cut) {
    if (!cut || head_size <= 0 || head_size % 32 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || n <= 0 || context <= 0 || max_len < 0 || window < 0 || sms <= 0) return B200_ERR_BAD_ARG;
    b200_kv4 kv;
    kv.head_size = head_size;
    kv.sms = sms;
    kv.view.context = context;
    kv.view.kv_heads = kv_heads;
    b200_kv4_attention_args a = {};
    a.n = n; a.heads = heads; a.max_len = max_len; a.window = window;
    const StepCut c = step_cut(&kv, a, quants != 0);
    cut[0] = c.heads; cut[1] = c.per_head; cut[2] = c.cluster; cut[3] = c.splits;
    return B200_OK;
}

int b200_log_probs(const b200_log_probs_args *a, void *stream, char *err, size_t err_len) {
    if (!a) return say(err, err_len, B200_ERR_BAD_ARG, "null arguments");
    if (a->rows < 0 || a->vocab <= 0) return say(err, err_len, B200_ERR_BAD_ARG, "%d rows of %d logits", a->rows, a->vocab);
    if (a->vocab > (1 << 30)) return say(err, err_len, B200_ERR_UNSUPPORTED, "%d logits a row (at most 2^30)", a->vocab);
    if (a->top < 0 || a->top > lp::MAX_TOP || a->top > a->vocab) return say(err, err_len, B200_ERR_BAD_ARG, "%d alternatives of %d logits (at most %d)", a->top, a->vocab, lp::MAX_TOP);
    if (!known_type(a->type)) return say(err, err_len, B200_ERR_UNSUPPORTED, "logits of type %d (FP32, FP16 and BF16 are known)", a->type);
    if (a->rows == 0) return B200_OK;
    if (!a->logits) return say(err, err_len, B200_ERR_BAD_ARG, "null logits");
    if (a->row_stride < a->vocab && a->rows > 1) return say(err, err_len, B200_ERR_BAD_ARG, "rows overlap: the stride is smaller than the row");
    if (a->rows > (1 << 26)) return say(err, err_len, B200_ERR_UNSUPPORTED, "too many rows in one call");
    OnDevice on(a->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess) e = log_probs_launch(*a, (cudaStream_t)stream);
    return e == cudaSuccess ? B200_OK : say(err, err_len, cuda_code(e), "%s", cudaGetErrorString(e));
}

} // extern "C"
