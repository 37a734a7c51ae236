// capi_kv.cu -- C ABI of the paged key/value cache and of the attention over it
// (include/hayai_cuda.h): the arguments' checks and the launches.
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

// The workspace of the engine's stream, or of the captures on it.
static int attn_workspace(hc_engine* e, AttnArgs* a) {
    cudaStreamCaptureStatus status;
    HC_CUDA(cudaStreamIsCapturing(e->stream, &status));
    const bool captured = status != cudaStreamCaptureStatusNone;
    AttnWs* w = e->attn_ws;
    while (w && (w->stream != e->stream || w->captured != captured)) w = w->next;
    if (!w) {
        // a capture forbids its thread to allocate unless it says that it means to, outside the graph
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        HC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        w = new (std::nothrow) AttnWs;
        const int rc = w ? attn_make_workspace(e, w) : hc_set_error(HC_ERR_CUDA, "attn_paged: out of host memory");
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (rc && w) {
            w->part.release();
            w->count.release();
            delete w;
        }
        if (rc) return rc;
        w->stream = e->stream;
        w->captured = captured;
        w->next = e->attn_ws;
        e->attn_ws = w;
    }
    a->part = (float*)w->part.p;
    a->count = (int*)w->count.p;
    return HC_OK;
}

extern "C" int hc_attn_paged_dev(hc_engine* e, const hc_kv_cache* c, const hc_kv_batch* b, int dtype, size_t n_heads,
                                 const void* q, size_t ldq, void* out, size_t ldo, float* lse, float scale, int causal,
                                 int window, int sink) {
    AttnArgs a{};
    int rc = hc_engine_activate(e);
    if (!rc) rc = check_cache(c, &a.c);
    if (!rc) rc = check_batch(e, c, b, &a.b);
    if (rc) return rc;
    if ((unsigned long long)b->n_tok * n_heads > INT32_MAX)
        return hc_set_error(HC_ERR_INVALID, "attn_paged: %d tokens of %zu heads are past 2^31 rows", b->n_tok, n_heads);
    if (n_heads == 0 || n_heads % (size_t)c->n_heads || n_heads > 65535)
        return hc_set_error(HC_ERR_INVALID, "attn_paged: %zu query heads on %d kv heads", n_heads, c->n_heads);
    if (window < 0 || sink < 0 || (window && !causal))
        return hc_set_error(HC_ERR_INVALID, "attn_paged: window %d and sink %d must not be negative, and a window needs causal",
                            window, sink);
    if (!isfinite(scale)) return hc_set_error(HC_ERR_INVALID, "attn_paged: scale is not finite");
    if (b->n_tok == 0 || b->n_seq == 0) return HC_OK;
    const size_t width = n_heads * c->head_dim;
    rc = check_rows("attn_paged", dtype, q, ldq, width);
    if (!rc) rc = check_rows("attn_paged", dtype, out, ldo, width);
    if (rc) return rc;
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.ldq = (long long)ldq;
    a.ldo = (long long)ldo;
    a.heads = (int)n_heads;
    a.group = (int)(n_heads / c->n_heads);
    a.by_group = FastDiv((uint32_t)a.group);
    a.by_page = FastDiv((uint32_t)c->page_size);
    a.causal = causal != 0;
    // no sequence holds more than 2^30 tokens, and positions less a window of that stay within 32 bits
    a.window = window < (1 << 30) ? window : 1 << 30;
    a.sink = window ? (sink < (1 << 30) ? sink : 1 << 30) : 0;
    a.scale = scale;
    const long long rows = (long long)(b->max_new && b->max_new < b->n_tok ? b->max_new : b->n_tok) * a.group;
    a.max_rows = (int)(rows < INT32_MAX ? rows : INT32_MAX);
    rc = attn_workspace(e, &a);
    if (rc) return rc;
    // Sequences of up to kFewRows rows per kv head go to the kernel for few rows (tiles of 8 or 16 rows), longer
    // ones to the other (tiles of 256): both are launched where the batch may have both.  At 16 rows, 16
    // sequences of 3000 to 8000 8-bit tokens take 67 us in the first and 145 in the second (bf16: 79 and
    // 113); at 32 rows, in tiles of 32, 182 and 147 (bf16: 115 and 116).
    constexpr int kFewRows = 16;
    const bool many = attn_many_supported(c->type, dtype) && a.max_rows > kFewRows;
    cudaError_t ce = cudaSuccess;
    if (many) {
        a.row_min = b->n_seq > 1 ? kFewRows + 1 : 1;
        a.row_max = INT32_MAX;
        ce = launch_attn_many(c->type, dtype, c->head_dim, a, e->num_sms, e->stream);
    }
    if (ce == cudaSuccess && (!many || b->n_seq > 1)) {
        a.row_min = 1;
        a.row_max = many ? kFewRows : INT32_MAX;
        if (many) a.max_rows = kFewRows;
        ce = launch_attn_few(c->type, dtype, c->head_dim, a, e->num_sms, e->stream);
    }
    return ce == cudaSuccess ? HC_OK : hc_cuda_error(ce, "attn_paged launch");
}
