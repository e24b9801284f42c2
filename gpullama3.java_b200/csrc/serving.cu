// serving.cu -- libb200llama.so: operators that serve many sequences from one pool of memory, and with drafted tokens (b200_paged_*, b200_verify_drafts): checks, cuts, launches.
#include "operators.h"
#include "operator_util.cuh"
#include "paged_chunk.cuh"
#include "verify.cuh"

#include <math.h>

namespace {

struct Fail { // the caller's message buffer
    char *err;
    size_t len;
    template <typename... A> int operator()(int code, const char *fmt, A... a) const { return say(err, len, code, fmt, a...); }
};

template <typename F> cudaError_t by_cache_type(int type, F &&f) { // f(a value of the type)
    if (type == B200_GGML_F16) return f(__half());
    return f(__nv_bfloat16());
}
int shift_of(int page_size) {
    int s = 0;
    while (1 << s < page_size) s++;
    return s;
}

int check_cache(const b200_paged_cache *c, const Fail &fail) {
    if (!c) return fail(B200_ERR_BAD_ARG, "null cache");
    if (c->type != B200_GGML_F16 && c->type != B200_GGML_BF16) return fail(B200_ERR_UNSUPPORTED, "a paged cache of type %d (FP16 and BF16 are known)", c->type);
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 96 && c->head_size != 128 && c->head_size != 256)
        return fail(B200_ERR_UNSUPPORTED, "a paged cache has heads of 32, 64, 96, 128 or 256 entries, not %d", c->head_size);
    if (c->pages <= 0 || c->kv_heads <= 0) return fail(B200_ERR_BAD_ARG, "pages and kv_heads must be positive");
    if (c->page_size < 1 || c->page_size > 65536 || (c->page_size & (c->page_size - 1))) return fail(B200_ERR_UNSUPPORTED, "pages hold a power of two of at most 65536 positions, not %d", c->page_size);
    if ((unsigned __int128)c->pages * c->kv_heads * c->page_size > 0xfffffff0u) return fail(B200_ERR_UNSUPPORTED, "a cache of more than 2^32 rows of a head");
    return B200_OK;
}
// positions, sequences and tables of a call
int check_rows(const b200_paged_cache *c, int n, const int32_t *positions, const int32_t *tables, int64_t table_stride, int n_sequences, int table_width, const Fail &fail) {
    if (n < 0) return fail(B200_ERR_BAD_ARG, "%d rows", n);
    if (n_sequences < 0 || table_width < 0 || (table_stride < table_width && n_sequences > 1)) return fail(B200_ERR_BAD_ARG, "%d tables of %d pages, %lld entries apart", n_sequences, table_width, (long long)table_stride);
    if ((long long)table_width * c->page_size > (1LL << 29)) return fail(B200_ERR_UNSUPPORTED, "a table of more than 2^29 positions");
    if (n && (!c->keys || !c->values)) return fail(B200_ERR_BAD_ARG, "null keys or values");
    if (reinterpret_cast<uintptr_t>(c->keys) % 16 || reinterpret_cast<uintptr_t>(c->values) % 16) return fail(B200_ERR_BAD_ARG, "keys and values have to start on 16-byte boundaries");
    if (n && (!positions || (!tables && n_sequences && table_width))) return fail(B200_ERR_BAD_ARG, "null positions or tables");
    return B200_OK;
}

struct Extent { // n rows of `width` bytes, `stride` bytes apart
    const void *at;
    __int128 stride, width;
    int n;
};
Extent pool_of(const b200_paged_cache *c, const void *at) { return {at, 0, (__int128)c->pages * c->kv_heads * c->page_size * c->head_size * 2, 1}; }
// Whether two such share a byte.  Rows of one stride may lie side by side, as parts of wider rows; others count as sharing where their extents do.
bool overlap(const Extent &x, const Extent &y) {
    const __int128 a = reinterpret_cast<uintptr_t>(x.at), b = reinterpret_cast<uintptr_t>(y.at);
    if (a + (x.n - 1) * x.stride + x.width <= b || b + (y.n - 1) * y.stride + y.width <= a) return false;
    if (x.n == 1 || y.n == 1 || x.stride != y.stride) return true;
    const __int128 d = ((b - a) % x.stride + x.stride) % x.stride; // where y's rows begin within x's
    return d < x.width || d + y.width > x.stride;
}

// How the attention of n rows is cut.
struct PagedCut {
    int nr, tokens, blocks, ctas; // blocks of 8 nr rows; tokens of a group; blocks of a group and key/value head; CTAs that units are shared out over (0: a CTA a unit)
    size_t units;
};
// Rows of a group: the tokens of a chunk that fit 32 rows (16 with heads of 256, for more their results would leave no registers), so that they read the pages once.
PagedCut paged_cut(const b200_paged_cache &c, const b200_paged_attention_args &a, int sms) {
    PagedCut k = {};
    const int G = c.kv_heads, mul = a.heads / G, chunk = a.chunk < 1 ? 1 : a.chunk < a.n ? a.chunk : a.n;
    int fit = (c.head_size == 256 ? 16 : 32) / mul;
    if (fit < 1) fit = 1;
    const int groups_of_chunk = (chunk + fit - 1) / fit;
    k.tokens = (chunk + groups_of_chunk - 1) / groups_of_chunk; // even shares
    // (a token of more than 16 query heads of a key/value head reads the pages once for 16 of them)
    k.nr = k.tokens > 1 ? (k.tokens * mul <= 16 ? 2 : (k.tokens * mul + 7) / 8) : mul <= 8 ? 1 : 2;
    k.blocks = (k.tokens * mul + 8 * k.nr - 1) / (8 * k.nr);
    const int KT = paged::step_keys(c.head_size), groups = (a.n + k.tokens - 1) / k.tokens;
    const long long context = (long long)a.table_width * c.page_size;
    long long len = a.max_len > 0 && a.max_len < context ? a.max_len : context;
    const long long near = (long long)a.window + k.tokens;
    if (a.window > 0 && near < len) len = near;
    k.units = (size_t)groups * G * k.blocks;
    // Shared out where the rows are long enough to pay for it (about 6 us: every CTA looks at all rows' positions, the parts are joined by a kernel of their own) and the units leave room.  us of a
    // captured call, a CTA a unit / shared out, by positions: one row of 8 heads of 128: 384: 8.3/10.1, 512: 9.7/10.8, 768: 12.8/11.0, 2048: 28.4/11.4; 8 rows of 8 heads of 64 (of room for 888 units):
    // 768: 10.3/11.4, 1024: 12.6/11.6, 2048: 21.6/12.7; 4 rows of a head of 256: 256: 11.4/11.1, 512: 17.7/11.4; 32 rows of 8 heads of 128 (256 units where 444 have room: no two CTAs for each) all of
    // one length: 1024: 27.5/34.7, 2048: 48.6/56.2; 24 rows of up to 4099: 74/49.  Three and four blocks of 8 rows, 8 heads, 16-bit results: 24 rows of 128: 320: 14.8/15.7, 384: 15.9/16.0, 512: 18.1/17.1, 1024: 27.2/17.3; 24 of
    // 64: 384: 11.9/13.7, 512: 13.4/14.4, 640: 15.1/14.7; 32 of 128: 256: 17.9/21.4, 320: 19.6/19.2, 512: 24.6/21.1; 32 of 64: 384: 13.9/15.4, 512: 15.8/16.3, 640: 17.7/16.4; 30 of 96: 384: 18.9/19.1, 448: 20.3/20.4, 512: 21.6/20.5; FP32
    // results, 24 of 128: 320: 17.4/17.4, 512: 22.5/19.3; 16 sequences (128 units for 444), 24 of 128: 768: 22.9/24.1, 1024: 28.5/27.9; 32 of 128: 640: 28.7/29.9, 768: 33.0/31.0; 32 of 64: 768: 19.7/21.5, 1024: 23.3/22.4.  Two of 128: 512:
    // 14.7/14.7, 640: 16.8/14.7.  (Half the positions of one or two blocks; between 340 and 600 heads of 64 lose up to 2 us.)
    const long long room = (long long)sms * paged::step_ctas(c.head_size, k.nr), units = (long long)k.units;
    const long long worth = (k.nr > 2 ? 10 : 20) * KT * (room + 4 * units) / room * (2 * units > room ? 2 : 1); // (a tile is latency, whatever the head's size)
    if (len > worth && groups <= paged::STEP_GROUPS && a.n <= paged::STEP_SHARED_ROWS) {
        const long long most = ((len + KT - 1) / KT + 1) * units / paged::SHARE_LEAST + 1;
        k.ctas = (int)(most < room ? most : room);
    }
    return k;
}
size_t paged_cut_bytes(const b200_paged_cache &c, const PagedCut &k) { return k.ctas ? (k.ctas + k.units) * 8 * k.nr * (c.head_size + 2) * 4 + (paged::STEP_GROUPS + 1) * 4 : 0; } // (paged::shared_grid)

// Chunks on tcgen05: 16-bit results, heads of 64, 96 or 128.  A tile takes 128 rows whether they are used or not.  us of a captured call in groups of 32 rows / as a chunk, by rows: 32/8 heads of 128, 8192
// positions: 64: 30.5/23.4, 128: 41.6/25.9, 512: 119/35; 1024 positions: 64: 22.9/19.3, 512: 33.5/20.9; 32/8 of 64, 8192: 64: 21.3/19.0; 16/16 of 64, 4096: 64: 23.9/18.7; 8/1 of 128, 8192: 64: 21.0/22.5,
// 128: 21.6/25.2, 512: 30.1/25.5 (the rule looks at a key/value head's rows alone: a few rows of a single head lose up to 4 us).
const int CHUNK_MIN_ROWS = 64;
struct PagedChunkCut {
    int tokens, splits;
    bool use;
};
PagedChunkCut paged_chunk_cut(const b200_paged_cache &c, const b200_paged_attention_args &a, int sms) {
    PagedChunkCut k = {};
    const int G = c.kv_heads, mul = a.heads / G, hs = c.head_size, chunk = a.chunk < a.n ? a.chunk : a.n;
    k.use = a.out_type != B200_GGML_F32 && (hs == 64 || hs == 96 || hs == 128) && mul <= paged::C_ROWS && chunk > 1 && (long long)chunk * mul >= CHUNK_MIN_ROWS;
    if (!k.use) return k;
    const int most = paged::C_ROWS / mul, shares = (chunk + most - 1) / most;
    k.tokens = (chunk + shares - 1) / shares; // even shares of a chunk: where all rows are chunks of that many tokens no CTA has two sequences' positions to run through
    const long long context = (long long)a.table_width * c.page_size, near = (long long)a.window + k.tokens;
    long long len = a.max_len > 0 && a.max_len < context ? a.max_len : context;
    if (a.window > 0 && near < len) len = near;
    const long long units = (long long)((a.n + k.tokens - 1) / k.tokens) * G, worth = len / (8 * paged::C_KEYS); // eight tiles of positions a CTA
    long long splits = sms / units;
    if (splits > worth) splits = worth;
    if (splits > paged::MAX_SPLITS) splits = paged::MAX_SPLITS;
    k.splits = splits < 1 ? 1 : (int)splits;
    return k;
}
size_t paged_work_bytes(const b200_paged_cache &c, const b200_paged_attention_args &a, int splits) { return splits > 1 ? (size_t)a.n * a.heads * splits * (c.head_size + 2) * 4 : 0; }
bool countable(const b200_paged_cache *c, const b200_paged_attention_args *a) {
    return c && a && a->n > 0 && a->heads > 0 && c->kv_heads > 0 && a->heads % c->kv_heads == 0 && a->table_width >= 0 && c->page_size > 0 && c->head_size > 0;
}

cudaError_t paged_attention_launch(const b200_paged_cache &c, const b200_paged_attention_args &a, cudaStream_t stream, bool give_up) {
    paged::Step k;
    k.pool = {c.keys, c.values, c.pages, c.kv_heads, shift_of(c.page_size)};
    k.rows = {a.positions, a.sequences, a.tables, a.table_stride, a.n, a.n_sequences, a.table_width * c.page_size};
    k.q = a.q; k.out = a.out;
    k.ldq = a.q_stride; k.ldo = a.out_stride;
    k.heads = a.heads; k.window = a.window; k.out_type = a.out_type;
    k.mul = a.heads / c.kv_heads;
    k.of = (65535 + k.mul) / k.mul;
    k.scale = a.scale;
    k.vec = aligned16(a.q, a.q_stride, 2);
    const int four = a.out_type == B200_GGML_F32 ? 16 : 8; // bytes of the four entries that a thread writes
    k.vec_out = reinterpret_cast<uintptr_t>(a.out) % four == 0 && a.out_stride % 4 == 0;
    k.work = (float *)a.workspace;
    const int sms = sm_count(c.device);
    const auto has_room = [&](int splits) { return a.workspace && paged_work_bytes(c, a, splits) <= a.workspace_bytes; };
    const auto join = [&](auto hs, int splits) { // a warp a row and head, a CTA where there are more parts than lanes
        const unsigned items = (unsigned)a.n * a.heads;
        if (splits <= 32) return launch(paged::k_paged_join_few<hs>, (items + 3) / 4, 128, 0, 1, true, stream, k);
        return launch(paged::k_paged_join<hs>, items, 128, 0, 1, true, stream, k);
    };
    if (PagedChunkCut cc = paged_chunk_cut(c, a, sms); cc.use) {
        if (!has_room(cc.splits)) cc.splits = 1;
        k.tokens = cc.tokens; k.splits = cc.splits;
        k.blocks = 1;
        k.ctas = 0;
        k.vec_out = aligned16(a.out, a.out_stride, 2);
        const unsigned grid = (unsigned)((a.n + cc.tokens - 1) / cc.tokens) * c.kv_heads * cc.splits;
        return by_cache_type(c.type, [&](auto type) {
            using T = decltype(type);
            const auto go = [&](auto hs) {
                constexpr size_t smem = paged::c_smem_bytes(hs);
                auto kern = paged::k_paged_chunk<hs, T>;
                if constexpr (hs == 64 && std::is_same<T, __half>::value) if (give_up) kern = paged::k_paged_chunk<hs, T, true>;
                cudaError_t e = allow_smem(kern, smem);
                if (e == cudaSuccess) e = launch(kern, grid, paged::C_THREADS, smem, 1, false, stream, k);
                return e != cudaSuccess || cc.splits == 1 ? e : join(hs, cc.splits);
            };
            if (c.head_size == 64) return go(std::integral_constant<int, 64>());
            if (c.head_size == 96) return go(std::integral_constant<int, 96>());
            return go(std::integral_constant<int, 128>());
        });
    }
    PagedCut cut = paged_cut(c, a, sms);
    if (!a.workspace || paged_cut_bytes(c, cut) > a.workspace_bytes) cut.ctas = 0;
    k.tokens = cut.tokens; k.blocks = cut.blocks; k.ctas = cut.ctas; k.splits = 1;
    const unsigned units = (unsigned)cut.units;
    return by_head_size(c.head_size, [&](auto hs) {
        return by_cache_type(c.type, [&](auto type) {
            using T = decltype(type);
            const auto go = [&](auto nr, auto lone) {
                constexpr size_t smem = paged::step_smem_bytes(hs, nr);
                auto kern = a.out_type == B200_GGML_F32 ? paged::k_paged_step<hs, T, nr, std::is_same<T, __half>::value ? 2 : 3, lone> : paged::k_paged_step<hs, T, nr, 1, lone>;
                cudaError_t e = allow_smem(kern, smem);
                if (e == cudaSuccess) e = launch(kern, cut.ctas ? cut.ctas + units : units, paged::STEP_WARPS * 32, smem, 1, false, stream, k);
                if (e != cudaSuccess || !cut.ctas) return e;
                if ((unsigned)cut.ctas <= 8 * units) return launch(paged::k_paged_join_shares<hs, nr, lone, true>, dim3(units, nr), 128, 0, 1, true, stream, k);
                return launch(paged::k_paged_join_shares<hs, nr, lone, false>, dim3(units, 8 * nr), 128, 0, 1, true, stream, k);
            };
            if (cut.tokens == 1) return cut.nr == 1 ? go(std::integral_constant<int, 1>(), std::true_type()) : go(std::integral_constant<int, 2>(), std::true_type());
            if constexpr (hs < 256) {
                if (cut.nr == 3) return go(std::integral_constant<int, 3>(), std::false_type());
                if (cut.nr == 4) return go(std::integral_constant<int, 4>(), std::false_type());
            }
            return go(std::integral_constant<int, 2>(), std::false_type());
        });
    });
}

int verify_stretches(int vocab) { return (vocab + verify::STRETCH - 1) / verify::STRETCH; }

} // namespace

extern "C" {

int b200_paged_append(const b200_paged_cache *c, const b200_paged_append_args *a, void *stream, char *err, size_t err_len) {
    const Fail fail = {err, err_len};
    int rc = check_cache(c, fail);
    if (rc) return rc;
    if (!a) return fail(B200_ERR_BAD_ARG, "null arguments");
    if ((rc = check_rows(c, a->n, a->positions, a->tables, a->table_stride, a->n_sequences, a->table_width, fail))) return rc;
    if (a->heads < 0) return fail(B200_ERR_BAD_ARG, "%d query heads", a->heads);
    if (!known_type(a->type)) return fail(B200_ERR_UNSUPPORTED, "rows of type %d (FP32, FP16 and BF16 are known)", a->type);
    if (a->rope_layout != B200_ROPE_HALF && a->rope_layout != B200_ROPE_INTERLEAVED) return fail(B200_ERR_BAD_ARG, "rotation layout %d", a->rope_layout);
    if (!a->cos != !a->sin) return fail(B200_ERR_BAD_ARG, "a rotation needs both tables");
    if (a->cos && (a->rope_dims <= 0 || a->rope_dims % 2 || a->rope_dims > c->head_size || a->rope_rows < 0)) return fail(B200_ERR_BAD_ARG, "a rotation of %d entries of %d, %d positions", a->rope_dims, c->head_size, a->rope_rows);
    if (a->n == 0) return B200_OK;
    if (!a->k || !a->v || (a->heads && (!a->q || !a->q_out))) return fail(B200_ERR_BAD_ARG, "null rows");
    const int64_t kv_width = (int64_t)c->kv_heads * c->head_size, q_width = (int64_t)a->heads * c->head_size;
    if (a->n > 1 && (a->k_stride < kv_width || a->v_stride < kv_width || (a->heads && (a->q_stride < q_width || a->q_out_stride < q_width)))) return fail(B200_ERR_BAD_ARG, "rows overlap: a stride is smaller than its row");
    if (a->heads + 2LL * c->kv_heads > (1LL << 18)) return fail(B200_ERR_UNSUPPORTED, "too many heads"); // (the grid's second dimension)
    if (a->heads) { // warps write q_out while others still read
        const int b = type_bytes(a->type);
        const Extent out = {a->q_out, (__int128)a->q_out_stride * 2, (__int128)q_width * 2, a->n}, q = {a->q, (__int128)a->q_stride * b, (__int128)q_width * b, a->n},
                     keys = {a->k, (__int128)a->k_stride * b, (__int128)kv_width * b, a->n}, values = {a->v, (__int128)a->v_stride * b, (__int128)kv_width * b, a->n};
        if (overlap(out, q) || overlap(out, keys) || overlap(out, values) || overlap(out, pool_of(c, c->keys)) || overlap(out, pool_of(c, c->values)))
            return fail(B200_ERR_BAD_ARG, "q_out may not overlap the rows or the cache");
    }
    paged::Append k;
    k.pool = {c->keys, c->values, c->pages, c->kv_heads, shift_of(c->page_size)};
    k.rows = {a->positions, a->sequences, a->tables, a->table_stride, a->n, a->n_sequences, a->table_width * c->page_size};
    if (a->cos && a->rope_rows < k.rows.context) k.rows.context = a->rope_rows; // (positions behind the tables' are padding)
    k.q = a->q; k.k = a->k; k.v = a->v;
    k.ldq = a->q_stride; k.ldk = a->k_stride; k.ldv = a->v_stride; k.ldo = a->q_out_stride;
    k.heads = a->heads;
    k.interleaved = a->rope_layout == B200_ROPE_INTERLEAVED;
    k.turned = a->cos ? a->rope_dims : 0;
    const int b = type_bytes(a->type);
    k.vec = aligned16(a->k, a->k_stride, b) && aligned16(a->v, a->v_stride, b) && (!a->heads || aligned16(a->q, a->q_stride, b));
    k.vec_out = !a->heads || aligned16(a->q_out, a->q_out_stride, 2);
    k.vec_tables = a->cos && a->rope_dims % 8 == 0 && aligned16(a->cos, 0, 4) && aligned16(a->sin, 0, 4); // rows of a multiple of 4 numbers
    k.q_norm = a->q_norm; k.k_norm = a->k_norm; k.cos = a->cos; k.sin = a->sin;
    k.eps = a->eps;
    k.q_out = a->q_out;
    OnDevice on(c->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess)
        e = by_head_size(c->head_size, [&](auto hs) {
            return by_type(a->type, [&](auto type) {
                return by_cache_type(c->type, [&](auto cache) {
                    constexpr int L = hs / 8, per_warp = L <= 4 ? 8 : L <= 8 ? 4 : L <= 16 ? 2 : 1;
                    const unsigned heads = (unsigned)(a->heads + 2 * c->kv_heads), per_cta = 8 * per_warp;
                    return launch(paged::k_paged_append<hs, decltype(type), decltype(cache)>, dim3((unsigned)a->n, (heads + per_cta - 1) / per_cta), 256, 0, 1, false, (cudaStream_t)stream, k);
                });
            });
        });
    return e == cudaSuccess ? B200_OK : fail(cuda_code(e), "%s", cudaGetErrorString(e));
}

size_t b200_paged_attention_workspace(const b200_paged_cache *c, const b200_paged_attention_args *a) {
    if (!countable(c, a)) return 0;
    const int sms = sm_count(c->device);
    const PagedChunkCut cc = paged_chunk_cut(*c, *a, sms);
    return cc.use ? paged_work_bytes(*c, *a, cc.splits) : paged_cut_bytes(*c, paged_cut(*c, *a, sms));
}

static int paged_attention(const b200_paged_cache *c, const b200_paged_attention_args *a, void *stream, char *err, size_t err_len, bool give_up) {
    const Fail fail = {err, err_len};
    int rc = check_cache(c, fail);
    if (rc) return rc;
    if (!a) return fail(B200_ERR_BAD_ARG, "null arguments");
    if ((rc = check_rows(c, a->n, a->positions, a->tables, a->table_stride, a->n_sequences, a->table_width, fail))) return rc;
    if (a->heads <= 0 || a->heads % c->kv_heads) return fail(B200_ERR_BAD_ARG, "%d query heads over %d key/value heads", a->heads, c->kv_heads);
    if (!known_type(a->out_type)) return fail(B200_ERR_UNSUPPORTED, "results of type %d (FP32, FP16 and BF16 are known)", a->out_type);
    if (a->window < 0 || a->max_len < 0 || a->chunk < 0) return fail(B200_ERR_BAD_ARG, "a negative window, length or chunk");
    if (!(fabsf(a->scale) < INFINITY)) return fail(B200_ERR_BAD_ARG, "a scale of %g", (double)a->scale);
    if (reinterpret_cast<uintptr_t>(a->workspace) % 16) return fail(B200_ERR_BAD_ARG, "the workspace is not aligned");
    if (a->n == 0) return B200_OK;
    if (!a->q || !a->out) return fail(B200_ERR_BAD_ARG, "null rows");
    const int64_t width = (int64_t)a->heads * c->head_size;
    if (a->n > 1 && (a->q_stride < width || a->out_stride < width)) return fail(B200_ERR_BAD_ARG, "rows overlap: a stride is smaller than its row");
    if ((long long)a->n * a->heads > (1LL << 27)) return fail(B200_ERR_UNSUPPORTED, "too many rows in one call");
    const int b = type_bytes(a->out_type);
    const Extent out = {a->out, (__int128)a->out_stride * b, (__int128)width * b, a->n}, q = {a->q, (__int128)a->q_stride * 2, (__int128)width * 2, a->n};
    const bool same = a->out == a->q && b == 2 && (a->n == 1 || a->out_stride == a->q_stride); // (a CTA reads the rows that it writes before it does)
    if ((!same && overlap(out, q)) || overlap(out, pool_of(c, c->keys)) || overlap(out, pool_of(c, c->values))) return fail(B200_ERR_BAD_ARG, "results may be the queries, but not overlap them or the cache otherwise");
    OnDevice on(c->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess) e = paged_attention_launch(*c, *a, (cudaStream_t)stream, give_up);
    return e == cudaSuccess ? B200_OK : fail(cuda_code(e), "%s", cudaGetErrorString(e));
}
int b200_paged_attention(const b200_paged_cache *c, const b200_paged_attention_args *a, void *stream, char *err, size_t err_len) { return paged_attention(c, a, stream, err, err_len, false); }
int b200_test_paged_give_up(const b200_paged_cache *c, const b200_paged_attention_args *a, void *stream, char *err, size_t err_len) {
    if (!countable(c, a) || c->head_size != 64 || c->type != B200_GGML_F16 || !paged_chunk_cut(*c, *a, 148).use) return say(err, err_len, B200_ERR_BAD_ARG, "no attention of a chunk with heads of 64 in FP16");
    return paged_attention(c, a, stream, err, err_len, true);
}

int b200_test_verify_weights(const float *x, int32_t n, float top, float temperature, double *weights) {
    if (n < 0 || (n && (!x || !weights)) || !(temperature >= 1e-4f && temperature <= 1e4f)) return B200_ERR_BAD_ARG;
    const double scale = verify::exp_scale(temperature);
    for (int32_t i = 0; i < n; i++) weights[i] = verify::exp_of(x[i], top, scale, [](int k) { return exp2((double)k / verify::EXP_TABLE); });
    return B200_OK;
}

int b200_test_verify_next(int32_t kind, const double *sums, double *rows) {
    if (kind < verify::TARGET || kind > verify::WHOLE || !sums || !rows) return B200_ERR_BAD_ARG;
    return verify::after_pass(kind, sums, rows[0], rows[1]);
}

size_t b200_verify_drafts_workspace(const b200_verify_drafts_args *a) {
    if (!a || a->sequences <= 0 || a->drafts < 0 || a->vocab <= 0) return 0;
    const size_t rows = (size_t)a->sequences * (a->drafts + 1) + (a->draft_logits && a->temperature != 0.0f ? (size_t)a->sequences * a->drafts : 0);
    return rows * verify_stretches(a->vocab) * sizeof(verify::Part);
}

int b200_verify_drafts(const b200_verify_drafts_args *a, void *stream, char *err, size_t err_len) {
    const Fail fail = {err, err_len};
    if (!a) return fail(B200_ERR_BAD_ARG, "null arguments");
    if (a->sequences < 0 || a->drafts < 0 || a->vocab <= 0) return fail(B200_ERR_BAD_ARG, "%d sequences, %d drafts, %d logits", a->sequences, a->drafts, a->vocab);
    if (a->drafts > verify::MAX_DRAFTS) return fail(B200_ERR_UNSUPPORTED, "%d drafts of a sequence (at most %d)", a->drafts, verify::MAX_DRAFTS);
    if (a->vocab > (1 << 24) || a->sequences > (1 << 16)) return fail(B200_ERR_UNSUPPORTED, "%d logits a row, %d sequences (at most 2^24, 2^16)", a->vocab, a->sequences);
    if (!known_type(a->type)) return fail(B200_ERR_UNSUPPORTED, "logits of type %d (FP32, FP16 and BF16 are known)", a->type);
    if (!(a->temperature == 0.0f || (a->temperature >= 1e-4f && a->temperature <= 1e4f))) return fail(B200_ERR_BAD_ARG, "a temperature of %g (0, or 1e-4 to 1e4)", (double)a->temperature);
    if (a->sequences == 0) return B200_OK;
    if (!a->logits || !a->out_tokens || !a->accepted || (a->drafts && !a->tokens) || (!a->uniforms && a->temperature != 0.0f)) return fail(B200_ERR_BAD_ARG, "a null argument");
    if (a->row_stride < a->vocab && a->drafts > 0) return fail(B200_ERR_BAD_ARG, "rows overlap: the stride is smaller than the row");
    const bool both = a->draft_logits && a->temperature != 0.0f && a->drafts > 0;
    const size_t need = b200_verify_drafts_workspace(a);
    if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16) return fail(B200_ERR_BAD_ARG, "a workspace of %zu bytes on a 16-byte boundary is needed", need);
    const __int128 S = a->sequences;
    const Extent drafts = {a->tokens, 0, S * a->drafts * 4, 1}, out = {a->out_tokens, 0, S * (a->drafts + 1) * 4, 1}, counts = {a->accepted, 0, S * 4, 1};
    if ((a->drafts && (overlap(out, drafts) || overlap(counts, drafts))) || overlap(out, counts)) return fail(B200_ERR_BAD_ARG, "results may not overlap the drafts or one another"); // (other sequences still read them)
    verify::Args k;
    k.logits = a->logits; k.draft_logits = both ? a->draft_logits : nullptr;
    k.ld_s = a->sequence_stride; k.ld_r = a->row_stride; k.draft_ld_s = a->draft_sequence_stride; k.draft_ld_r = a->draft_row_stride;
    k.sequences = a->sequences; k.drafts = a->drafts; k.vocab = a->vocab;
    k.stretches = verify_stretches(a->vocab);
    const int b = type_bytes(a->type);
    k.vec = aligned16(a->logits, a->sequence_stride, b) && (a->drafts == 0 || a->row_stride * b % 16 == 0) &&
            (!both || (aligned16(a->draft_logits, a->draft_sequence_stride, b) && a->draft_row_stride * b % 16 == 0));
    k.temperature = a->temperature;
    k.greedy = a->temperature == 0.0f; k.both = both;
    k.tokens = a->tokens; k.uniforms = a->uniforms; k.out_tokens = a->out_tokens; k.accepted = a->accepted;
    k.parts = (verify::Part *)a->workspace;
    const unsigned long long grid = (unsigned long long)a->sequences * (a->drafts + 1 + (both ? a->drafts : 0)) * k.stretches;
    if (grid > 0x7fffffffull) return fail(B200_ERR_UNSUPPORTED, "too many logits in one call");
    OnDevice on(a->device);
    cudaError_t e = on.error;
    if (e == cudaSuccess)
        e = by_type(a->type, [&](auto type) {
            using T = decltype(type);
            const cudaError_t first = launch(verify::k_verify_rows<T>, (unsigned)grid, verify::ROW_THREADS, 0, 1, false, (cudaStream_t)stream, k);
            if (first == cudaSuccess && k.greedy) return launch(verify::k_verify_greedy, (unsigned)a->sequences, 256, 0, 1, true, (cudaStream_t)stream, k);
            return first != cudaSuccess ? first : launch(verify::k_verify_token<T>, (unsigned)a->sequences * verify::CLUSTER, verify::TOKEN_THREADS, 0, verify::CLUSTER, true, (cudaStream_t)stream, k);
        });
    return e == cudaSuccess ? B200_OK : fail(cuda_code(e), "%s", cudaGetErrorString(e));
}

} // extern "C"
