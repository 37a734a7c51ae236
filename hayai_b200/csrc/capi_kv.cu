// capi_kv.cu -- C ABI of the paged key/value cache, its bookkeeping, rotary positions and the attention
// over it (include/hayai_cuda.h): the arguments' checks and the launches.
#include <math.h>

#include <new>

#include "../../include/hayai_cuda.h"
#include "engine.h"
#include "kv_launch.h"

using namespace hc;

static_assert(HC_KV_MAX_SEQ == HC_KV_SEQS, "one limit");

static bool half_type(int t) { return t == T_F16 || t == T_BF16; }

static int check_cache(const hc_kv_cache* c, KvDev* d) {
    if (!c) return hc_set_error(HC_ERR_INVALID, "null cache");
    if (!half_type(c->type) && c->type != T_I8)
        return hc_set_error(HC_ERR_UNSUPPORTED, "kv cache: no kernel for type %d (f16, bf16 or i8)", c->type);
    if (c->head_dim != 64 && c->head_dim != 128)
        return hc_set_error(HC_ERR_UNSUPPORTED, "kv cache: head_dim %d (64 or 128)", c->head_dim);
    if (c->n_pages < 1 || c->page_size < 1 || c->n_heads < 1)
        return hc_set_error(HC_ERR_INVALID, "kv cache: empty shape n_pages=%d n_heads=%d page_size=%d", c->n_pages,
                            c->n_heads, c->page_size);
    if (!c->k || !c->v || (c->type == T_I8 && (!c->k_scale || !c->v_scale)))
        return hc_set_error(HC_ERR_INVALID, "kv cache: null %s", c->k && c->v ? "scales" : "pages");
    const size_t es = c->type == T_I8 ? 1 : 2;
    const size_t st[3] = {c->page_stride, c->head_stride, c->row_stride}, n[3] = {(size_t)c->n_pages, (size_t)c->n_heads,
                                                                                 (size_t)c->page_size};
    size_t last = 0;
    for (int i = 0; i < 3; ++i) {
        if (st[i] * es % 64 || st[i] < (size_t)c->head_dim)
            return hc_set_error(HC_ERR_INVALID, "kv cache: stride %zu must be a multiple of 64 bytes and no less than head_dim",
                                st[i]);
        if (st[i] > ((size_t)1 << 38) / n[i])
            return hc_set_error(HC_ERR_INVALID, "kv cache: stride %zu reaches past 256 GiB", st[i]);
        last += st[i] * (n[i] - 1);
    }
    if (last * es / 64 > UINT32_MAX) return hc_set_error(HC_ERR_INVALID, "kv cache: the strides reach past 256 GiB");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15)
        return hc_set_error(HC_ERR_INVALID, "kv cache: pages must be 16-byte aligned");
    if (c->type == T_I8 && c->scale_page_stride < (size_t)c->n_heads * c->page_size)
        return hc_set_error(HC_ERR_INVALID, "kv cache: scale page stride %zu < n_heads * page_size", c->scale_page_stride);
    d->k = (uint8_t*)c->k;
    d->v = (uint8_t*)c->v;
    d->ks = c->k_scale;
    d->vs = c->v_scale;
    d->page = (uint32_t)(c->page_stride * es / 64);
    d->head = (uint32_t)(c->head_stride * es / 64);
    d->row = (uint32_t)(c->row_stride * es / 64);
    d->spage = (long long)c->scale_page_stride;
    d->n_pages = c->n_pages;
    d->page_size = c->page_size;
    d->n_heads = c->n_heads;
    return HC_OK;
}

static int check_batch(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, KvBatchDev* d) {
    if (!b) return hc_set_error(HC_ERR_INVALID, "null batch");
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_pages < 0 || b->max_new < 0)
        return hc_set_error(HC_ERR_INVALID, "kv batch: negative size n_seq=%d n_tok=%d max_new=%d max_pages=%d", b->n_seq,
                            b->n_tok, b->max_new, b->max_pages);
    if (b->n_seq > HC_KV_MAX_SEQ)
        return hc_set_error(HC_ERR_INVALID, "kv batch: %d sequences (at most %d)", b->n_seq, HC_KV_MAX_SEQ);
    if ((long long)b->max_pages * c->page_size > (1 << 30))
        return hc_set_error(HC_ERR_INVALID, "kv batch: %d pages of %d reach past 2^30 tokens", b->max_pages, c->page_size);
    if (b->n_tok > 0 && b->n_seq > 0 && (!b->page_table || !b->q_start || !b->kv_len))
        return hc_set_error(HC_ERR_INVALID, "kv batch: null page table, q_start or kv_len");
    if (b->table_stride < (size_t)b->max_pages)
        return hc_set_error(HC_ERR_INVALID, "kv batch: table stride %zu < max_pages %d", b->table_stride, b->max_pages);
    d->table = b->page_table;
    d->table_stride = (long long)b->table_stride;
    d->q_start = b->q_start;
    d->kv_len = b->kv_len;
    d->n_seq = b->n_seq;
    d->n_tok = b->n_tok;
    d->max_pages = b->max_pages;
    d->err = e->d_err;
    return HC_OK;
}

static size_t elem_bytes(int dtype) { return dtype == T_F32 ? 4 : 2; }

// A packed row array [n_tok][heads * head_dim] of f32, f16 or bf16 with leading dimension ld.
static int check_rows(const char* what, int dtype, const void* p, size_t ld, size_t width) {
    if (dtype != T_F32 && !half_type(dtype))
        return hc_set_error(HC_ERR_UNSUPPORTED, "%s: no kernel for rows of type %d (f32, f16 or bf16)", what, dtype);
    if (!p) return hc_set_error(HC_ERR_INVALID, "%s: null rows", what);
    if (ld < width) return hc_set_error(HC_ERR_INVALID, "%s: leading dimension %zu smaller than the row length %zu", what, ld, width);
    if (((uintptr_t)p & 15) || ld * elem_bytes(dtype) % 16)
        return hc_set_error(HC_ERR_INVALID, "%s: rows must be 16-byte aligned with a leading dimension of whole 16 bytes", what);
    return HC_OK;
}

static int kv_rows(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, const void* k, size_t ldk,
                   const void* v, size_t ldv, bool write) {
    const char* what = write ? "kv_append" : "kv_read";
    KvDev cd;
    KvBatchDev bd;
    int rc = hc_engine_activate(e);
    if (!rc) rc = check_cache(c, &cd);
    if (!rc) rc = check_batch(e, c, b, &bd);
    if (rc) return rc;
    const size_t width = (size_t)c->n_heads * c->head_dim;
    if (b->n_tok == 0 || b->n_seq == 0) return HC_OK;
    rc = check_rows(what, dtype, k, ldk, width);
    if (!rc) rc = check_rows(what, dtype, v, ldv, width);
    if (rc) return rc;
    const KvRows r{(void*)k, (void*)v, (long long)ldk, (long long)ldv};
    const cudaError_t ce = write ? launch_kv_append(c->type, dtype, c->head_dim, cd, bd, r, e->stream)
                                 : launch_kv_read(c->type, dtype, c->head_dim, cd, bd, r, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, write ? "kv_append launch" : "kv_read launch");
}

extern "C" int hc_kv_append_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, const void* k,
                                size_t ldk, const void* v, size_t ldv) {
    return kv_rows(e, c, b, dtype, k, ldk, v, ldv, true);
}

extern "C" int hc_kv_read_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, void* k, size_t ldk,
                              void* v, size_t ldv) {
    return kv_rows(e, c, b, dtype, k, ldk, v, ldv, false);
}

// A new workspace, as much as any call of any kernel takes, so that it never moves under a captured graph.  Its
// counters are zero before any stream gets it.
static int attn_make_workspace(const hc_engine* e, AttnWs* w) {
    int rc = w->part.ensure(kAttnPartBytes * e->num_sms);
    if (!rc) rc = w->count.ensure((size_t)e->num_sms * 32 * sizeof(int));  // one for each row of a block's first split tile
    if (rc) return rc;
    HC_CUDA(cudaMemsetAsync(w->count.p, 0, w->count.cap, cudaStreamPerThread));
    HC_CUDA(cudaStreamSynchronize(cudaStreamPerThread));
    return HC_OK;
}

// The workspace of the engine's stream, or of the captures on it, with `base` bytes for a shared prefix; *base_at is null
// where there is no room for those.
static int attn_workspace(hc_engine* e, AttnArgs* a, size_t base, void** base_at) {
    cudaStreamCaptureStatus status;
    HC_CUDA(cudaStreamIsCapturing(e->stream, &status));
    const bool captured = status != cudaStreamCaptureStatusNone;
    AttnWs* w = e->attn_ws;
    while (w && (w->stream != e->stream || w->captured != captured || (captured && w->base.cap < base))) w = w->next;
    if (!w || w->base.cap < base) {
        // a power of two, past 256 MB in quarters: it grows few times, and takes little more than it needs where that is much
        size_t size = base ? (size_t)1 << 20 : 0;
        while (size < base) size *= 2;
        if (const size_t step = size / 8; size > (size_t)256 << 20)
            while (size - step >= base) size -= step;
        // a capture forbids its thread to allocate unless it says that it means to, outside the graph
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        HC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        const bool fresh = !w;
        size_t left = SIZE_MAX, all;
        // an allocation that fails ends a capture: not to be tried where there is no room for it
        if (captured && base && cudaMemGetInfo(&left, &all) == cudaSuccess && left < size + 2 * kAttnPartBytes * e->num_sms) {
            cudaThreadExchangeStreamCaptureMode(&mode);
            return attn_workspace(e, a, 0, base_at);
        }
        if (fresh) w = new (std::nothrow) AttnWs;
        int rc = !w ? hc_set_error(HC_ERR_CUDA, "attn_paged: out of host memory") : fresh ? attn_make_workspace(e, w) : HC_OK;
        if (!rc && size) rc = w->base.ensure(size);  // (freeing what was there waits for the calls that use it)
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (rc && w && fresh) {
            w->part.release();
            w->count.release();
            delete w;
        }
        if (rc) {
            cudaGetLastError();  // reported here: the next launch's check is not to find it
            return base ? attn_workspace(e, a, 0, base_at) : rc;
        }
        if (fresh) {
            w->stream = e->stream;
            w->captured = captured;
            w->next = e->attn_ws;
            e->attn_ws = w;
        }
    }
    a->part = (float*)w->part.p;
    a->count = (int*)w->count.p;
    if (base_at) *base_at = base ? w->base.p : nullptr;
    return HC_OK;
}

// What the attention calls have in common: their checks, and the arguments that both kernels get.  *none: nothing to do.
static int attn_args(const char* what, hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, size_t n_heads,
                     const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale, AttnArgs* a, bool* none) {
    int rc = hc_engine_activate(e);
    if (!rc) rc = check_cache(c, &a->c);
    if (!rc) rc = check_batch(e, c, b, &a->b);
    if (rc) return rc;
    if ((unsigned long long)b->n_tok * n_heads > INT32_MAX)
        return hc_set_error(HC_ERR_INVALID, "%s: %d tokens of %zu heads are past 2^31 rows", what, b->n_tok, n_heads);
    if (n_heads == 0 || n_heads % (size_t)c->n_heads || n_heads > 65535)
        return hc_set_error(HC_ERR_INVALID, "%s: %zu query heads on %d kv heads", what, n_heads, c->n_heads);
    if (!isfinite(scale)) return hc_set_error(HC_ERR_INVALID, "%s: scale is not finite", what);
    *none = b->n_tok == 0 || b->n_seq == 0;
    if (*none) return HC_OK;
    const size_t width = n_heads * c->head_dim;
    rc = check_rows(what, dtype, q, ldq, width);
    if (!rc) rc = check_rows(what, dtype, out, ldo, width);
    if (rc) return rc;
    a->q = q;
    a->out = out;
    a->lse = lse;
    a->ldq = (long long)ldq;
    a->ldo = (long long)ldo;
    a->heads = (int)n_heads;
    a->group = (int)(n_heads / c->n_heads);
    a->by_group = FastDiv((uint32_t)a->group);
    a->by_page = FastDiv((uint32_t)c->page_size);
    a->causal = 1;
    a->scale = scale;
    return HC_OK;
}

// Whether sharing is worth it where the program gives no bound.  Readings of a prefix by tiles of rows are counted, alone
// and together; the figures are us in a graph, paged and shared, of one group, 32 heads on 8 of 128, prefixes not in L2.
// A bound has two sides: the host's, for what the page tables could hold at most, and the device's for what there is, which
// is lower as the call has paid for the plan by then (9 to 12 us, where nothing is shared after all).
struct ShareBound {
    long long host, device;
};
// Single tokens (16-bit rows) pay for several kernels' starts, and for a prefix's units more than for a reading of it: as much
// as for one more from 16-bit pages and three more from 8-bit ones.  bf16 pages: 4 sequences behind 16384 (192 MB saved) 36 and
// 45, 16 behind 4096 (240) 36 and 42, 8 behind 16384 (448) 59 and 48, 40 behind 4096 (624) 72 and 56, 16 behind 16384 (960) 102
// and 53, 4 behind 65536 (768) 160 and 79.  8-bit: 16 behind 4096 (124 MB) 33 and 47, 8 behind 16384 (231) 52 and 53, 40 behind
// 4096 (322) 66 and 59, 16 behind 16384 (495) 90 and 62; 4 behind 65536 (396) 90 and 94, 8 (924) 165 and 102.
constexpr ShareBound kShareBytes{300 << 20, 200 << 20}, kShareBytes8{190 << 20, 120 << 20};
// Chunks have starts of the same cost either way.  Where they are fewer tiles than blocks, the paged attention splits tiles,
// and whatever is read again can be saved: 8 of 5 tokens behind 1024 (28 MB) 37 and 36, 16 of 5 behind 1024 (60 MB) 44 and 45, 4
// behind 4096 (48 MB) 45 and 37, 16 of 64 behind 4096 (240 MB) 141 and 136, 8 behind 16384 (448 MB) 215 and 178.  With more,
// what counts is tiles that sharing fills, against its own tiles at 27/25 of the others' time and 16 bytes for each of
// the rows' values in pieces: 16 of 256 tokens behind 16384 (960 MB, no tile saved) 1075 and 1281, 8 of 1000 (448 MB, 3 of 128)
// 2342 and 2499, 16 of 100 (7 of 32) behind 16384 556 and 490, behind 1024 111 and 125; one of 3000 with 31 single tokens behind
// 1024 265 and 337, behind 16384 1101 and 1044.
constexpr ShareBound kShareChunkBytes{64 << 20, 32 << 20};
// f32 rows read a prefix by up to 16 of them, which costs 8/5 of a reading by up to 8; in tokens of a kv head at the cheaper
// one, less 48 of them for moving a row's parts (500 tokens and 63 single ones behind 1024: 249 and 308, behind 4096 679 and 619).
// 8-bit pages: 16 sequences of 2 tokens behind 16384 (0.42 M saved) 120 and 136, 8 single tokens (0.63 M) 62 and 75, 40 behind
// 4096 (0.79 M) 81 and 85, 8 of 5 behind 16384 (1.26 M) 178 and 155, 16 single ones (1.26 M) 114 and 94; bf16 pages, 8 (0.63 M) 85 and
// 86, 40 behind 4096 (0.79 M) 107 and 93, 16 (1.26 M) 157 and 114.  16 tokens save nothing: 16 behind 16384 661 and 712.
constexpr ShareBound kShareTokens{700000, 500000}, kShareTokens8{1000000, 750000};

// Sequences with up to kFewRows rows per kv head go to the kernel for few rows (tiles of 8 or 16 rows), longer
// ones to the other (tiles of 256): both are launched where the batch may have both.  At 16 rows, 16
// sequences of 3000 to 8000 8-bit tokens take 67 us in the first and 145 in the second (bf16: 79 and
// 113); at 32 rows, in tiles of 32, 182 and 147 (bf16: 115 and 116).
static cudaError_t attn_run(const hc_engine* e, const hc_kv_cache* c, int dtype, AttnArgs a, int max_new) {
    const long long rows = (long long)(max_new && max_new < a.b.n_tok ? max_new : a.b.n_tok) * a.group;
    a.max_rows = (int)(rows < INT32_MAX ? rows : INT32_MAX);
    const bool many = attn_many_supported(c->type, dtype) && a.max_rows > kFewRows;
    cudaError_t ce = cudaSuccess;
    if (many) {
        a.row_min = a.b.n_seq > 1 ? kFewRows + 1 : 1;
        a.row_max = INT32_MAX;
        ce = launch_attn_many(c->type, dtype, c->head_dim, a, e->num_sms, e->stream);
    }
    if (ce == cudaSuccess && (!many || a.b.n_seq > 1)) {
        a.row_min = 1;
        a.row_max = many ? kFewRows : INT32_MAX;
        if (many) a.max_rows = kFewRows;
        ce = launch_attn_few(c->type, dtype, c->head_dim, a, e->num_sms, e->stream);
    }
    return ce;
}

extern "C" int hc_attn_paged_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, size_t n_heads,
                                 const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale, int causal,
                                 int window, int sink) {
    AttnArgs a{};
    bool none;
    if (window < 0 || sink < 0 || (window && !causal))
        return hc_set_error(HC_ERR_INVALID, "attn_paged: window %d and sink %d must not be negative, and a window needs causal",
                            window, sink);
    int rc = attn_args("attn_paged", e, c, b, dtype, n_heads, q, ldq, out, ldo, lse, scale, &a, &none);
    if (rc || none) return rc;
    a.causal = causal != 0;
    // no sequence holds more than 2^30 tokens, and positions less a window of that stay within 32 bits
    a.window = window < (1 << 30) ? window : 1 << 30;
    a.sink = window ? (sink < (1 << 30) ? sink : 1 << 30) : 0;
    rc = attn_workspace(e, &a, 0, nullptr);
    if (rc) return rc;
    const cudaError_t ce = attn_run(e, c, dtype, a, b->max_new);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "attn_paged launch");
}

extern "C" int hc_attn_shared_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, const hc_kv_shared* g, int dtype,
                                  size_t n_heads, const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale) {
    AttnArgs a{};
    bool none;
    int rc = attn_args("attn_shared", e, c, b, dtype, n_heads, q, ldq, out, ldo, lse, scale, &a, &none);
    if (rc) return rc;
    if (!g) return hc_set_error(HC_ERR_INVALID, "attn_shared: null groups");
    if (g->n_groups < 0 || g->max_new < 0 || g->least < 0)
        return hc_set_error(HC_ERR_INVALID, "attn_shared: negative size n_groups=%d max_new=%d least=%lld", g->n_groups, g->max_new,
                            (long long)g->least);
    if (g->n_groups > HC_KV_MAX_SEQ)
        return hc_set_error(HC_ERR_INVALID, "attn_shared: %d groups (at most %d)", g->n_groups, HC_KV_MAX_SEQ);
    if (g->n_groups && (!g->seq_start || !g->length)) return hc_set_error(HC_ERR_INVALID, "attn_shared: null seq_start or length");
    if (none) return HC_OK;
    // f32 rows go to the kernel for few rows, whose terms attn_prefix.cu's operands do not hold, in two calls.
    const int sms = e->num_sms;
    const bool few = !attn_many_supported(c->type, dtype), codes = c->type == T_I8;
    const long long rows = (long long)b->n_tok * (long long)n_heads, kv = c->n_heads;
    const long long own_rows = (long long)(b->max_new && b->max_new < b->n_tok ? b->max_new : b->n_tok) * a.group;
    // Sharing is left where what it saves is not worth its kernels: here where the page tables do not reach so far, else by
    // the groups' lengths and rows, on the device.
    const long long token = 2 * kv * (c->head_dim * (codes ? 1 : 2) + (codes ? 4 : 0));
    KvSharedDev d{};
    d.rule = g->least == 0;
    d.tile = few ? 16 : 256;
    d.extra = codes ? 3 : 1;
    d.alone = own_rows > 8 ? 8 : 5;
    d.chunk = kShareChunkBytes.device / token;
    d.moved = few ? rows * 48 / kv : rows * c->head_dim * 16 / token;
    const ShareBound bound = few ? (codes ? kShareTokens8 : kShareTokens) : codes ? kShareBytes8 : kShareBytes;
    d.least = g->least ? g->least : bound.device / (few ? kv : token);
    // the most that the sequences save, in fifths of readings of all that their tables hold
    long long readings = 5 * (b->n_seq - 1ll), least = g->least;
    const long long new_rows = (long long)b->n_tok * a.group;
    if (d.rule && few) {
        least = bound.host / kv;
        readings = d.alone * (long long)b->n_seq - 8 * (d.alone == 8 ? 1 : (new_rows + 15) / 16);
    } else if (d.rule && new_rows > (long long)kFewRows * b->n_seq) {  // one chunk at least
        least = kShareChunkBytes.host / token;
    } else if (d.rule) {
        least = bound.host / token;
        readings -= 5 * d.extra;
    }
    const bool may = g->n_groups && b->n_tok >= 2 && readings * b->max_pages * c->page_size / 5 >= least;
    // What a sequence has behind its prefix goes there too where it has few rows (single tokens) and makes more than a block's
    // tile, or two of 16-bit pages: us of calls behind 16384 tokens, 32 heads on 8 of 128, as tiles of attn_prefix.cu and
    // there, 16 sequences with 50 tokens of their own each (128 tiles), 8-bit 62 and 66, bf16 54 and 63; with 1000 75 and 78, 66 and
    // 78; 24 with 1000 89 and 86, 76 and 91; 36 with 50 (288) 85 and 76, 69 and 68; 64 with 50 116 and 82, 91 and 77, with
    // 3000 260 and 163, 172 and 206; 128 with 50 199 and 107, 153 and 96.
    const long long seqs = b->n_seq < b->n_tok ? b->n_seq : b->n_tok;  // with new tokens
    const bool behind = few || (own_rows <= kFewRows && seqs * kv > (codes ? 1 : 2) * sms);
    long long shared = b->n_seq / 2;  // groups that share anything: two sequences with new tokens each
    if (shared > b->n_tok / 2) shared = b->n_tok / 2;
    if (shared > g->n_groups) shared = g->n_groups;
    const long long tiles = 2 * (rows / 256) + (few ? 0 : shared * kv) + (behind ? seqs : seqs * kv);
    // a row's result in a piece (of narrow tiles two) of its prefix, and one behind it unless it comes from the kernel
    // for few rows; and where a block's share ends in a tile, its rows once more
    auto narrow = [&](long long n) { return n * kv * 128 < rows ? n * kv * 128 : rows; };
    const long long pieces =
        few ? 0 : rows + narrow(shared) + (behind ? 0 : rows + narrow(seqs)) + (long long)sms * 256;
    size_t size = 0;
    auto room = [&](size_t n) {
        const size_t at = size;
        size += (n * 4 + 255) / 256 * 256;
        return at;
    };
    const size_t r_few = few ? (size_t)rows : 0, r_behind = behind ? (size_t)rows : 0;
    const size_t at_first = room(HC_KV_SEQS), at_q = room(HC_KV_SEQS + 1), at_len = room(HC_KV_SEQS), at_row = room(HC_KV_SEQS),
                 at_line = room(kLineInts), at_block = room((size_t)sms), at_tiles = room((size_t)tiles * sizeof(PrefixTile) / 4),
                 at_lse = room(r_behind), at_out = room(r_behind * c->head_dim), at_flse = room(r_few), at_few = room(r_few * c->head_dim),
                 at_ml = room((size_t)pieces * 2), at_part = room((size_t)pieces * c->head_dim);
    void* base = nullptr;
    rc = attn_workspace(e, &a, may ? size : 0, &base);
    if (rc) return rc;
    if (!base) {  // nothing can be shared, or there is no room for it
        const cudaError_t ce = attn_run(e, c, dtype, a, b->max_new);
        return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "attn_shared launch");
    }
    auto place = [&](size_t at) { return (void*)((uint8_t*)base + at); };
    d.seq_start = g->seq_start;
    d.length = g->length;
    d.n = g->n_groups;
    d.first = (int*)place(at_first);
    d.q_start = (int*)place(at_q);
    d.len = (int*)place(at_len);
    d.row = (int*)place(at_row);
    d.heads = a.heads;
    d.kv_heads = c->n_heads;
    d.few = few;
    d.few_behind = behind;
    d.blocks = sms;
    d.max_tiles = (int)(tiles < INT32_MAX ? tiles : INT32_MAX);
    d.max_pieces = (int)(pieces < INT32_MAX ? pieces : INT32_MAX);
    d.tiles = (PrefixTile*)place(at_tiles);
    d.line = (int*)place(at_line);
    d.first_tile = (int*)place(at_block);
    cudaError_t ce = launch_attn_groups(a.b, d, b->max_pages * c->page_size, e->stream);
    AttnArgs plain = a;  // the paged attention, where nothing is shared after all
    plain.unless = d.line + kLineTiles;
    plain.shared = plain.early = 1;
    PrefixArgs p{d.tiles, d.line, d.first_tile, (float*)place(at_part), (float*)place(at_ml), nullptr, nullptr};
    AttnArgs x = a;  // of the kernel for few rows
    x.shared = 1;
    x.only = d.line + kLineTiles;
    x.row_min = 1;
    x.row_max = INT32_MAX;
    if (few) {
        AttnArgs y = x;
        y.b.q_start = d.q_start;
        y.b.kv_len = d.len;
        y.b.n_seq = d.n;
        y.table_row = d.row;
        y.causal = 0;
        y.to_base = 1;
        y.base = (float*)place(at_few);
        y.base_lse = (float*)place(at_flse);
        const long long most = (long long)(g->max_new && g->max_new < b->n_tok ? g->max_new : b->n_tok) * a.group;
        y.max_rows = (int)(most < INT32_MAX ? most : INT32_MAX);
        p.few = y.base;
        p.few_lse = y.base_lse;
        if (ce == cudaSuccess) ce = launch_attn_few(c->type, dtype, c->head_dim, y, sms, e->stream);
    } else if (ce == cudaSuccess) {
        ce = launch_attn_prefix(c->type, dtype, c->head_dim, a, p, sms, e->stream);
    }
    if (behind) {
        x.first = d.first;
        x.base = a.base = (float*)place(at_out);
        x.base_lse = a.base_lse = (float*)place(at_lse);
        x.early = 1;
        x.max_rows = (int)(own_rows < INT32_MAX ? own_rows : INT32_MAX);
        if (ce == cudaSuccess) ce = launch_attn_few(c->type, dtype, c->head_dim, x, sms, e->stream);
    }
    if (ce == cudaSuccess) ce = launch_attn_join(dtype, c->head_dim, a, p, sms, e->stream);
    if (ce == cudaSuccess) ce = attn_run(e, c, dtype, plain, b->max_new);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "attn_shared launch");
}

// ------------------------------------------------------------------ rotary positions
static int check_rope(const hc_rope* r, RopeDev* d) {
    if (!r) return hc_set_error(HC_ERR_INVALID, "null rope");
    if (r->layout != HC_ROPE_HALF && r->layout != HC_ROPE_PAIRS)
        return hc_set_error(HC_ERR_INVALID, "rope: layout %d (HC_ROPE_HALF or HC_ROPE_PAIRS)", r->layout);
    if (r->head_dim < 2 || r->head_dim > 2 * HC_ROPE_MAX || r->head_dim % 2 || r->rot_dim < 2 || r->rot_dim % 2 ||
        r->rot_dim > r->head_dim)
        return hc_set_error(HC_ERR_INVALID, "rope: rot_dim %d of head_dim %d (even, at most %d)", r->rot_dim, r->head_dim,
                            2 * HC_ROPE_MAX);
    if (!isfinite(r->amplitude)) return hc_set_error(HC_ERR_INVALID, "rope: amplitude is not finite");
    d->pairs = r->layout == HC_ROPE_PAIRS;
    d->dim = r->head_dim;
    d->rot = r->rot_dim;
    d->amplitude = r->amplitude;
    for (int i = 0; i < r->rot_dim / 2; ++i) d->turns[i] = r->turns[i];
    return HC_OK;
}
// Are values turned in chunks of 8, or of 8 and their 8 partners?
static bool rope_chunks(const RopeDev& r) { return r.dim % 16 == 0 && r.rot % (r.pairs ? 8 : 16) == 0; }

extern "C" int hc_rope_init(hc_rope* out, int layout, int head_dim, int rot_dim, double base, double factor, double original,
                            double low, double high, const float* factors, float amplitude) {
    if (!out) return hc_set_error(HC_ERR_INVALID, "null out pointer");
    hc_rope r{};
    r.layout = layout;
    r.head_dim = head_dim;
    r.rot_dim = rot_dim ? rot_dim : head_dim;
    r.amplitude = amplitude;
    RopeDev unused;
    const int rc = check_rope(&r, &unused);
    if (rc) return rc;
    if (!(base > 0) || !isfinite(base) || !(factor > 0) || !isfinite(factor))
        return hc_set_error(HC_ERR_INVALID, "rope: base %g and factor %g must be positive", base, factor);
    if (!(original >= 0) || !isfinite(original) || (original > 0 && !(low < high && isfinite(low) && isfinite(high))))
        return hc_set_error(HC_ERR_INVALID, "rope: original context %g must not be negative, and needs low < high (%g, %g)",
                            original, low, high);
    const long double tau = 6.283185307179586476925286766559L;
    for (int i = 0; i < r.rot_dim / 2; ++i) {
        if (factors && (!(factors[i] > 0) || !isfinite(factors[i])))
            return hc_set_error(HC_ERR_INVALID, "rope: factors must be positive");
        long double t = powl((long double)base, -2.0L * i / r.rot_dim) / (factors ? factors[i] : 1.0L);
        if (original > 0) {
            long double g = ((long double)original * t / tau - low) / ((long double)high - low);
            g = g < 0 ? 0 : g > 1 ? 1 : g;
            t *= (1 - g) / factor + g;
        } else {
            t /= factor;
        }
        const long double turn = t / tau;  // whole turns make no difference
        if (!(turn < 0x1p62L)) return hc_set_error(HC_ERR_INVALID, "rope: frequency %d is out of range", i);
        const long double part = roundl((turn - floorl(turn)) * 0x1p64L);
        r.turns[i] = part >= 0x1p64L ? 0 : (uint64_t)part;
    }
    *out = r;
    return HC_OK;
}

// Are they the same rows?
static bool rows_same(const void* x, size_t ldx, const void* out, size_t ldo, size_t n) { return x == out && (ldx == ldo || n == 1); }
// May rows be written at `out` while rows are read at `x`?  Where both are the same rows, or no row of the one touches
// a row of the other (slices of one array's rows, or apart altogether).
static bool rows_apart(const void* x, size_t ldx, size_t wx, const void* out, size_t ldo, size_t wo, size_t n, size_t es) {
    const uint64_t a = (uint64_t)(uintptr_t)x, b = (uint64_t)(uintptr_t)out;
    if (n == 0 || a + ((n - 1) * ldx + wx) * es <= b || b + ((n - 1) * ldo + wo) * es <= a) return true;
    if (ldx != ldo) return false;
    const uint64_t pitch = ldx * es, off = b >= a ? (b - a) % pitch : (pitch - (a - b) % pitch) % pitch;
    return off >= wx * es && off + wo * es <= pitch;
}

extern "C" int hc_rope_dev(hc_engine* e, const hc_rope* rope, int dtype, size_t n_tok, size_t n_heads, const int32_t* positions,
                           const void* x, size_t ldx, void* out, size_t ldo) {
    RopeDev r{};
    int rc = hc_engine_activate(e);
    if (!rc) rc = check_rope(rope, &r);
    if (rc) return rc;
    if (dtype != T_F32 && !half_type(dtype))
        return hc_set_error(HC_ERR_UNSUPPORTED, "rope: no kernel for rows of type %d (f32, f16 or bf16)", dtype);
    if (n_tok > INT32_MAX || n_heads > 65535 || n_tok * n_heads > INT32_MAX)
        return hc_set_error(HC_ERR_INVALID, "rope: %zu tokens of %zu heads are past 2^31 rows", n_tok, n_heads);
    if (n_tok == 0 || n_heads == 0) return HC_OK;
    if (!positions || !x || !out) return hc_set_error(HC_ERR_INVALID, "rope: null positions or rows");
    const size_t width = n_heads * r.dim, es = elem_bytes(dtype);
    if (ldx < width || ldo < width || ldx > ((size_t)1 << 40) || ldo > ((size_t)1 << 40))
        return hc_set_error(HC_ERR_INVALID, "rope: leading dimension %zu out of range for rows of %zu", ldx < width ? ldx : ldo, width);
    if (((uintptr_t)x | (uintptr_t)out) % es) return hc_set_error(HC_ERR_INVALID, "rope: rows are not aligned to their type");
    if (!rows_same(x, ldx, out, ldo, n_tok) && !rows_apart(x, ldx, width, out, ldo, width, n_tok, es))
        return hc_set_error(HC_ERR_INVALID, "rope: out must be x itself or not overlap it");
    const bool wide = rope_chunks(r) && (((uintptr_t)x | (uintptr_t)out) & 15) == 0 && ldx * es % 16 == 0 && ldo * es % 16 == 0;
    const RopeRows a{positions, x, out, (long long)ldx, (long long)ldo, (int)n_tok, (int)n_heads};
    const cudaError_t ce = launch_rope(dtype, r, a, wide, e->num_sms, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "rope launch");
}

extern "C" int hc_kv_append_rope_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, const hc_rope* rope, int dtype,
                                     size_t n_heads, const void* q, size_t ldq, void* q_out, size_t ldqo, const void* k,
                                     size_t ldk, const void* v, size_t ldv) {
    const char* what = "kv_append_rope";
    KvDev cd;
    KvBatchDev bd;
    RopeDev r{};
    int rc = hc_engine_activate(e);
    if (!rc) rc = check_cache(c, &cd);
    if (!rc) rc = check_batch(e, c, b, &bd);
    if (!rc) rc = check_rope(rope, &r);
    if (rc) return rc;
    if (r.dim != c->head_dim)
        return hc_set_error(HC_ERR_INVALID, "%s: the rope's head_dim is %d, the cache's %d", what, r.dim, c->head_dim);
    if (!rope_chunks(r))
        return hc_set_error(HC_ERR_UNSUPPORTED, "%s: rot_dim %d (a multiple of 16, in pairs of 8; hc_rope_dev takes the others)",
                            what, r.rot);
    if (n_heads == 0 || n_heads > 65535 || c->n_heads > 65535 ||
        (unsigned long long)b->n_tok * (n_heads + 2ull * c->n_heads) > INT32_MAX)
        return hc_set_error(HC_ERR_INVALID, "%s: %d tokens of %zu query and %d kv heads", what, b->n_tok, n_heads, c->n_heads);
    if (b->n_tok == 0 || b->n_seq == 0) return HC_OK;
    const size_t width = n_heads * c->head_dim, kw = (size_t)c->n_heads * c->head_dim, es = elem_bytes(dtype), n = b->n_tok;
    rc = check_rows(what, dtype, q, ldq, width);
    if (!rc) rc = check_rows(what, dtype, q_out, ldqo, width);
    if (!rc) rc = check_rows(what, dtype, k, ldk, kw);
    if (!rc) rc = check_rows(what, dtype, v, ldv, kw);
    if (rc) return rc;
    if ((!rows_same(q, ldq, q_out, ldqo, n) && !rows_apart(q, ldq, width, q_out, ldqo, width, n, es)) ||
        !rows_apart(k, ldk, kw, q_out, ldqo, width, n, es) || !rows_apart(v, ldv, kw, q_out, ldqo, width, n, es))
        return hc_set_error(HC_ERR_INVALID, "%s: q_out must be q itself or overlap neither q, k nor v", what);
    const RopeAppend a{q, k, v, q_out, (long long)ldq, (long long)ldqo, (long long)ldk, (long long)ldv, (int)n_heads};
    const cudaError_t ce = launch_kv_append_rope(c->type, dtype, c->head_dim, r, cd, bd, a, e->num_sms, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "kv_append_rope launch");
}

// ------------------------------------------------------------------ the cache's bookkeeping
extern "C" int hc_kv_pages_scratch(int n_pages, size_t* out) {
    if (!out || n_pages < 1) return hc_set_error(HC_ERR_INVALID, "kv pages: n_pages %d, or a null pointer", n_pages);
    *out = kv_pages_scratch(n_pages);
    return HC_OK;
}

// The pages' description, and its layers by kMaxLayers (room for `most` such groups).
static int check_pages(const char* what, hc_engine* e, const hc_kv_pages* p, PagesDev* d, KvLayers* layers, int most, int* groups) {
    int rc = hc_engine_activate(e);
    if (rc) return rc;
    if (!p) return hc_set_error(HC_ERR_INVALID, "%s: null pages", what);
    if (p->n_layers < 1 || !p->layers) return hc_set_error(HC_ERR_INVALID, "%s: no layers", what);
    if (p->n_layers > most * kMaxLayers)
        return hc_set_error(HC_ERR_INVALID, "%s: %d layers (at most %d)", what, p->n_layers, most * kMaxLayers);
    const hc_kv_cache* const c0 = p->layers;
    for (int i = 0; i < p->n_layers; ++i) {
        const hc_kv_cache* const c = p->layers + i;
        KvDev k;
        rc = check_cache(c, &k);
        if (rc) return rc;
        if (c->type != c0->type || c->n_pages != c0->n_pages || c->n_heads != c0->n_heads || c->page_size != c0->page_size ||
            c->head_dim != c0->head_dim || c->page_stride != c0->page_stride || c->head_stride != c0->head_stride ||
            c->row_stride != c0->row_stride || c->scale_page_stride != c0->scale_page_stride)
            return hc_set_error(HC_ERR_INVALID, "%s: layer %d has another shape than the first", what, i);
        KvLayers& y = layers[i / kMaxLayers];
        const int at = i % kMaxLayers;
        y.k[at] = k.k;
        y.v[at] = k.v;
        y.ks[at] = c->type == T_I8 ? k.ks : nullptr;
        y.vs[at] = c->type == T_I8 ? k.vs : nullptr;
        if (at == 0) {
            y.page = k.page;
            y.head = k.head;
            y.row = k.row;
            y.spage = k.spage;
            y.n_heads = c->n_heads;
            y.row_bytes = c->head_dim * (c->type == T_I8 ? 1 : 2);
        }
        y.n = at + 1;
    }
    *groups = (p->n_layers + kMaxLayers - 1) / kMaxLayers;
    if (p->n_slots < 0 || p->max_pages < 0)
        return hc_set_error(HC_ERR_INVALID, "%s: negative size n_slots=%d max_pages=%d", what, p->n_slots, p->max_pages);
    if ((long long)p->max_pages * c0->page_size > (1 << 30))
        return hc_set_error(HC_ERR_INVALID, "%s: %d pages of %d reach past 2^30 tokens", what, p->max_pages, c0->page_size);
    if (c0->page_size > 1 << 26)  // a warp's copy counts a head's rows of a page, 16 bytes at a time, in 32 bits
        return hc_set_error(HC_ERR_UNSUPPORTED, "%s: pages of %d tokens (at most 2^26)", what, c0->page_size);
    if (p->n_slots && (!p->page_table || !p->kv_len))
        return hc_set_error(HC_ERR_INVALID, "%s: null page table or kv_len", what);
    if (!p->refs || !p->scratch) return hc_set_error(HC_ERR_INVALID, "%s: null refs or scratch", what);
    if (p->table_stride < (size_t)p->max_pages)
        return hc_set_error(HC_ERR_INVALID, "%s: table stride %zu < max_pages %d", what, p->table_stride, p->max_pages);
    d->table = p->page_table;
    d->stride = (long long)p->table_stride;
    d->len = p->kv_len;
    d->refs = p->refs;
    d->n_slots = p->n_slots;
    d->max_pages = p->max_pages;
    d->n_pages = c0->n_pages;
    d->page_size = c0->page_size;
    d->by_page = FastDiv((uint32_t)c0->page_size);
    const size_t moves = d->n_pages > HC_KV_SEQS ? d->n_pages : HC_KV_SEQS;
    d->moves = p->scratch;
    d->item = d->moves + 16;
    d->src = d->item + 4 * HC_KV_SEQS;
    d->dst = d->src + moves;
    d->rows = d->dst + moves;
    d->free = d->rows + moves;
    d->err = e->d_err;
    return HC_OK;
}
constexpr int kLayerGroups = 4;

static int check_items(const char* what, int n, const void* a, const void* b) {
    if (n < 0 || n > HC_KV_MAX_SEQ) return hc_set_error(HC_ERR_INVALID, "%s: %d sequences (at most %d)", what, n, HC_KV_MAX_SEQ);
    if (n && (!a || !b)) return hc_set_error(HC_ERR_INVALID, "%s: null array", what);
    return HC_OK;
}

extern "C" int hc_kv_fork_dev(hc_engine* e, const hc_kv_pages* p, int n, const int32_t* parents, const int32_t* children) {
    PagesDev d{};
    KvLayers y[kLayerGroups];
    int groups = 0, rc = check_pages("kv_fork", e, p, &d, y, kLayerGroups, &groups);
    if (!rc) rc = check_items("kv_fork", n, parents, children);
    if (rc || n == 0) return rc;
    const cudaError_t ce = launch_kv_fork(d, y, groups, n, parents, children, e->num_sms, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "kv_fork launch");
}

extern "C" int hc_kv_resize_dev(hc_engine* e, const hc_kv_pages* p, int n, const int32_t* slots, const int32_t* lens) {
    PagesDev d{};
    KvLayers y[kLayerGroups];
    int groups = 0, rc = check_pages("kv_resize", e, p, &d, y, kLayerGroups, &groups);
    if (!rc) rc = check_items("kv_resize", n, slots, lens);
    if (rc || n == 0) return rc;
    const cudaError_t ce = launch_kv_resize(d, y, groups, n, slots, lens, e->num_sms, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "kv_resize launch");
}

extern "C" int hc_kv_compact_dev(hc_engine* e, const hc_kv_pages* p, int32_t* moved) {
    PagesDev d{};
    KvLayers y[kLayerGroups];
    int groups = 0;
    const int rc = check_pages("kv_compact", e, p, &d, y, kLayerGroups, &groups);
    if (rc) return rc;
    const cudaError_t ce = launch_kv_compact(d, y, groups, moved, e->num_sms, e->stream);
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "kv_compact launch");
}
