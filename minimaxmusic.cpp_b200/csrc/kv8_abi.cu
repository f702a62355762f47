// kv8_abi.cu - C ABI of the 8-bit paged KV cache (the mm3fa_kv8_* part of include/mm3fa.h).
//
// Checks the descriptors, fills the launch parameters and enqueues on the caller's stream; nothing
// allocates device memory or synchronises.
#include "../../include/mm3fa.h"
#include "kv8.cuh"

#include <algorithm>
#include <cmath>
#include <cstdint>

using namespace mm3fa;

namespace {

bool aligned_to(const void * p, size_t a) {
    return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

int64_t elem_bytes(int t) {
    return t == MM3FA_TYPE_F32 ? 4 : (t == MM3FA_TYPE_F16 || t == MM3FA_TYPE_BF16) ? 2 : 0;
}

int check_cache(const mm3fa_kv8 * c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
        return MM3FA_ERR_NULL;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (c->n_head_kv < 1 || c->n_pages < 1 || c->n_layers < 1 || c->reserved != 0) {
        return MM3FA_ERR_SHAPE;
    }
    if (c->n_head_kv > 32767) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4)) {
        return MM3FA_ERR_ALIGN;
    }
    return MM3FA_OK;
}

int check_table(const mm3fa_kv8 * c, const mm3fa_kv8_table * t) {
    if (!t || !t->pages) {
        return MM3FA_ERR_NULL;
    }
    if (t->n_seq < 1 || t->max_pages < 1 || t->stride < t->max_pages) {
        return MM3FA_ERR_SHAPE;
    }
    // token positions are 32-bit; sequences are a grid dimension
    if (t->n_seq > 65535 || (int64_t) t->max_pages * c->page_tokens > INT32_MAX) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    return aligned_to(t->pages, 4) ? MM3FA_OK : MM3FA_ERR_ALIGN;
}

// The attention rounds token counts up to its blocks and looks some ahead, in 32 bits.
bool attn_tokens_fit(const mm3fa_kv8 * c, const mm3fa_kv8_table * t) {
    return (int64_t) t->max_pages * c->page_tokens <= (int64_t) 1 + INT32_MAX - 8192;
}

// Rows [D, ne1, ne2, ne3] of a floating type; strides are any multiples of the element size.
int check_rows(const mm3fa_tensor * t, int64_t D) {
    if (!t) {
        return MM3FA_ERR_NULL;
    }
    const int64_t e = elem_bytes(t->type);
    if (e == 0) {
        return MM3FA_ERR_TYPE;
    }
    if (t->ne[0] != D || t->ne[1] < 1 || t->ne[2] < 1 || t->ne[3] < 1) {
        return MM3FA_ERR_SHAPE;
    }
    if (!t->data) {
        return MM3FA_ERR_NULL;
    }
    if ((int64_t) t->nb[0] != e || t->nb[1] % e || t->nb[2] % e || t->nb[3] % e) {
        return MM3FA_ERR_STRIDE;
    }
    return aligned_to(t->data, (size_t) e) ? MM3FA_OK : MM3FA_ERR_ALIGN;
}

// Rows that are written: no two of them may share bytes through a stride below a row's.
int check_out(const mm3fa_tensor * t, int64_t D) {
    const int st = check_rows(t, D);
    if (st != MM3FA_OK) {
        return st;
    }
    for (int i = 1; i < 4; i++) {
        if (t->ne[i] > 1 && (int64_t) t->nb[i] < D * elem_bytes(t->type)) {
            return MM3FA_ERR_STRIDE;
        }
    }
    return MM3FA_OK;
}

Kv8Rows rows_of(const mm3fa_tensor * t) {
    Kv8Rows r{};
    r.data = static_cast<char *>(t->data);
    r.nb1  = (int64_t) t->nb[1];
    r.nb2  = (int64_t) t->nb[2];
    r.nb3  = (int64_t) t->nb[3];
    r.type = t->type;
    r.vec  = aligned_to(t->data, 16) && (t->ne[1] == 1 || t->nb[1] % 16 == 0) && (t->ne[2] == 1 || t->nb[2] % 16 == 0) &&
            (t->ne[3] == 1 || t->nb[3] % 16 == 0);
    return r;
}

Kv8Layer layer_of(const mm3fa_kv8 * c, int layer) {
    Kv8Layer      l{};
    const int64_t heads = (int64_t) layer * c->n_pages * c->n_head_kv, page = (int64_t) c->page_tokens * c->head_dim;
    l.k         = c->k + heads * page;
    l.v         = c->v + heads * page;
    l.k_scale   = c->k_scale + heads;
    l.v_scale   = c->v_scale + heads;
    l.n_pages   = c->n_pages;
    l.n_head_kv = c->n_head_kv;
    l.D         = c->head_dim;
    l.P         = c->page_tokens;
    for (l.log2p = 0; (1 << l.log2p) < l.P; l.log2p++) {
    }
    return l;
}

Kv8Table table_of(const mm3fa_kv8_table * t) {
    Kv8Table r{};
    r.pages     = t->pages;
    r.stride    = t->stride;
    r.max_pages = t->max_pages;
    r.n_seq     = t->n_seq;
    return r;
}

int check_store(const mm3fa_kv8 * c, int layer, const mm3fa_tensor * k, const mm3fa_tensor * v, const mm3fa_kv8_table * t,
                const int32_t * start) {
    int st = check_cache(c);
    if (st == MM3FA_OK) {
        st = check_table(c, t);
    }
    if (st == MM3FA_OK && !start) {
        st = MM3FA_ERR_NULL;
    }
    if (st == MM3FA_OK && (layer < 0 || layer >= c->n_layers)) {
        st = MM3FA_ERR_SHAPE;
    }
    for (const mm3fa_tensor * x : { k, v }) {
        if (st == MM3FA_OK) {
            st = check_rows(x, c->head_dim);
        }
        if (st == MM3FA_OK && (x->ne[1] != k->ne[1] || x->ne[2] != c->n_head_kv || x->ne[3] != t->n_seq)) {
            st = MM3FA_ERR_SHAPE;
        }
    }
    if (st == MM3FA_OK && k->ne[1] > (1 << 30)) {
        st = MM3FA_ERR_UNSUPPORTED;
    }
    return st;
}

Kv8StoreParams store_params(const mm3fa_kv8 * c, int layer, const mm3fa_tensor * k, const mm3fa_tensor * v,
                            const mm3fa_kv8_table * t, const int32_t * start, const int32_t * n) {
    Kv8StoreParams p{};
    p.c      = layer_of(c, layer);
    p.t      = table_of(t);
    p.k      = rows_of(k);
    p.v      = rows_of(v);
    p.start  = start;
    p.n      = n;
    p.n_rows = (int) k->ne[1];
    return p;
}

size_t pages_workspace(const mm3fa_kv8 * c, int64_t n_seq) {
    return std::max(KV8_WS_ZEROED, 4 * ((size_t) KV8_WS_HEAD + 3 * (size_t) c->n_pages + 2 * (size_t) n_seq));
}

// The workspace's parts; MM3FA_ERR_WORKSPACE where it is missing, too small or not 4-byte aligned.
int plan_workspace(const mm3fa_kv8 * c, const mm3fa_kv8_table * t, void * ws, size_t bytes, Kv8PlanParams & p) {
    const int n_seq = t->n_seq;
    if ((int64_t) n_seq * t->max_pages > INT32_MAX) {  // the pages that a call needs are counted in 32 bits
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (!ws || bytes < pages_workspace(c, n_seq) || !aligned_to(ws, 4)) {
        return MM3FA_ERR_WORKSPACE;
    }
    p.status   = static_cast<uint32_t *>(ws);
    p.head     = static_cast<int *>(ws);
    p.copy_src = p.head + KV8_WS_HEAD;
    p.copy_dst = p.copy_src + c->n_pages;
    p.map      = p.copy_dst + c->n_pages;
    p.win      = p.map + c->n_pages;
    p.off      = p.win + n_seq;
    p.n_pages  = c->n_pages;
    p.P        = c->page_tokens;
    return MM3FA_OK;
}

Kv8PoolCopy pool_copy(const mm3fa_kv8 * c) {
    Kv8PoolCopy r{};
    r.k          = reinterpret_cast<char *>(c->k);
    r.v          = reinterpret_cast<char *>(c->v);
    r.k_scale    = c->k_scale;
    r.v_scale    = c->v_scale;
    r.n_layers   = c->n_layers;
    r.n_pages    = c->n_pages;
    r.n_head_kv  = c->n_head_kv;
    r.page_bytes = (int64_t) c->n_head_kv * c->page_tokens * c->head_dim;
    return r;
}

// A table's entries, from its first to its last, as a byte range.
bool tables_overlap(const mm3fa_kv8_table * a, const mm3fa_kv8_table * b) {
    const int32_t * a0 = a->pages, *a1 = a0 + (a->n_seq - 1) * a->stride + a->max_pages;
    const int32_t * b0 = b->pages, *b1 = b0 + (b->n_seq - 1) * b->stride + b->max_pages;
    return a0 < b1 && b0 < a1;
}

bool ranges_overlap(const int32_t * a, const int32_t * b, int64_t n) {
    return a < b + n && b < a + n;
}

int check_tables_out(const mm3fa_kv8 * c, const mm3fa_kv8_table * in, const int32_t * refs_in, const mm3fa_kv8_table * out,
                     const int32_t * refs_out) {
    int st = check_cache(c);
    if (st == MM3FA_OK) {
        st = check_table(c, in);
    }
    if (st == MM3FA_OK) {
        st = check_table(c, out);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (!refs_in || !refs_out) {
        return MM3FA_ERR_NULL;
    }
    if (in->n_seq != out->n_seq || in->max_pages != out->max_pages) {
        return MM3FA_ERR_SHAPE;
    }
    // results go to buffers of their own: a sequence may be read as a source after it was replaced
    if (tables_overlap(in, out) || ranges_overlap(refs_in, refs_out, c->n_pages)) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    return aligned_to(refs_in, 4) && aligned_to(refs_out, 4) ? MM3FA_OK : MM3FA_ERR_ALIGN;
}

}  // namespace

extern "C" {

int mm3fa_kv8_append(const mm3fa_kv8 * cache, int layer, const mm3fa_tensor * k_new, const mm3fa_tensor * v_new,
                     const mm3fa_kv8_table * table, const int32_t * start, const int32_t * n_new, void * stream) {
    const int st = check_store(cache, layer, k_new, v_new, table, start);
    if (st != MM3FA_OK) {
        return st;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    return host_record_cuda(launch_kv8_append(store_params(cache, layer, k_new, v_new, table, start, n_new),
                                              static_cast<cudaStream_t>(stream)));
}

int mm3fa_kv8_read(const mm3fa_kv8 * cache, int layer, const mm3fa_kv8_table * table, const int32_t * start,
                   const int32_t * n, mm3fa_tensor * k_out, mm3fa_tensor * v_out, void * stream) {
    int st = check_store(cache, layer, k_out, v_out, table, start);
    for (const mm3fa_tensor * x : { (const mm3fa_tensor *) k_out, (const mm3fa_tensor *) v_out }) {
        if (st == MM3FA_OK) {
            st = check_out(x, cache->head_dim);
        }
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    return host_record_cuda(launch_kv8_read(store_params(cache, layer, k_out, v_out, table, start, n), static_cast<cudaStream_t>(stream)));
}

size_t mm3fa_kv8_attn_workspace(const mm3fa_kv8 * cache, const mm3fa_tensor * q, const mm3fa_kv8_table * table) {
    if (!q || check_cache(cache) != MM3FA_OK || check_table(cache, table) != MM3FA_OK || !attn_tokens_fit(cache, table) || q->ne[1] < 1 || q->ne[2] < 1 ||
        q->ne[2] % cache->n_head_kv || q->ne[1] > (1 << 24) || q->ne[2] > (1 << 20) ||
        q->ne[2] / cache->n_head_kv * q->ne[1] > (1 << 24)) {
        return 0;
    }
    return std::max(KV8_WS_ZEROED, kv8_attn_workspace_bytes(cache->head_dim, q->ne[1] * (q->ne[2] / cache->n_head_kv),
                                                            (int64_t) cache->n_head_kv * table->n_seq,
                                                            (int64_t) table->max_pages * cache->page_tokens, host_sm_count()));
}

int mm3fa_kv8_attn(const mm3fa_kv8 * cache, int layer, const mm3fa_tensor * q, const mm3fa_kv8_table * table,
                   const int32_t * kv_len, const int32_t * q_len, float scale, float logit_softcap, int causal,
                   mm3fa_tensor * dst, void * workspace, size_t workspace_bytes, void * stream) {
    int st = check_cache(cache);
    if (st == MM3FA_OK) {
        st = check_table(cache, table);
    }
    if (st == MM3FA_OK) {
        st = check_rows(q, cache->head_dim);
    }
    if (st == MM3FA_OK) {
        st = check_out(dst, cache->head_dim);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (!kv_len) {
        return MM3FA_ERR_NULL;
    }
    if (dst->type != MM3FA_TYPE_F32 && dst->type != q->type) {
        return MM3FA_ERR_TYPE;
    }
    const int64_t H = q->ne[2];
    if (layer < 0 || layer >= cache->n_layers || H % cache->n_head_kv || q->ne[3] != table->n_seq || dst->ne[1] != H ||
        dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3] || !std::isfinite(scale) || !(logit_softcap >= 0.0f) ||
        !std::isfinite(logit_softcap)) {
        return MM3FA_ERR_SHAPE;
    }
    // rows of a kv head, and 32-key blocks of all rows at the table's full length, are counted in 32 bits
    const int64_t rows = H / cache->n_head_kv * q->ne[1];
    if (!attn_tokens_fit(cache, table) || q->ne[1] > (1 << 24) || H > (1 << 20) || rows > (1 << 24) || rows * (H / cache->n_head_kv) > INT32_MAX ||
        ((rows + 15) / 16) * cache->n_head_kv * table->n_seq > (int64_t) INT32_MAX / (((int64_t) table->max_pages * cache->page_tokens + 31) / 32)) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < mm3fa_kv8_attn_workspace(cache, q, table)) {
        return MM3FA_ERR_WORKSPACE;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    Kv8AttnParams p{};
    p.c          = layer_of(cache, layer);
    p.t          = table_of(table);
    p.q          = rows_of(q);
    p.o          = rows_of(dst);
    p.kv_len     = kv_len;
    p.q_len      = q_len;
    p.n_q        = (int) q->ne[1];
    p.n_head     = (int) H;
    p.ratio      = (int) (H / cache->n_head_kv);
    p.causal     = causal != 0;
    p.scale      = scale;
    p.softcap    = logit_softcap;
    p.status     = static_cast<uint32_t *>(workspace);
    p.timeout_ns = host_wait_timeout_ns();
    return host_record_cuda(launch_kv8_attn(p, host_sm_count(), static_cast<cudaStream_t>(stream)));
}

size_t mm3fa_kv8_pages_workspace(const mm3fa_kv8 * cache, int n_seq) {
    return check_cache(cache) == MM3FA_OK && n_seq >= 1 ? pages_workspace(cache, n_seq) : 0;
}

int mm3fa_kv8_reserve(const mm3fa_kv8 * cache, mm3fa_kv8_table * table, int32_t * refs, const int32_t * n_tok,
                      void * workspace, size_t workspace_bytes, void * stream) {
    int st = check_cache(cache);
    if (st == MM3FA_OK) {
        st = check_table(cache, table);
    }
    if (st == MM3FA_OK && (!refs || !n_tok)) {
        st = MM3FA_ERR_NULL;
    }
    Kv8PlanParams p{};
    if (st == MM3FA_OK) {
        st = plan_workspace(cache, table, workspace, workspace_bytes, p);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    p.table_out  = const_cast<int32_t *>(table->pages);
    p.out_stride = table->stride;
    p.n_seq      = table->n_seq;
    p.max_pages  = table->max_pages;
    p.refs_out   = refs;
    p.n_tok      = n_tok;
    return host_record_cuda(launch_kv8_reserve(p, static_cast<cudaStream_t>(stream)));
}

int mm3fa_kv8_fork(const mm3fa_kv8 * cache, const mm3fa_kv8_table * table, const int32_t * kv_len, const int32_t * refs,
                   const int32_t * src, const int32_t * dst, int n_pairs, uint32_t flags, mm3fa_kv8_table * table_out,
                   int32_t * kv_len_out, int32_t * refs_out, void * workspace, size_t workspace_bytes, void * stream) {
    int st = check_tables_out(cache, table, refs, table_out, refs_out);
    if (st == MM3FA_OK && (!kv_len || !kv_len_out || (n_pairs > 0 && !dst))) {
        st = MM3FA_ERR_NULL;
    }
    if (st == MM3FA_OK && n_pairs < 0) {
        st = MM3FA_ERR_SHAPE;
    }
    if (st == MM3FA_OK && ((flags & ~(uint32_t) MM3FA_KV8_FORK_DEEP) || ranges_overlap(kv_len, kv_len_out, table->n_seq))) {
        st = MM3FA_ERR_UNSUPPORTED;
    }
    Kv8PlanParams p{};
    if (st == MM3FA_OK) {
        st = plan_workspace(cache, table, workspace, workspace_bytes, p);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    p.table_in   = table->pages;
    p.table_out  = const_cast<int32_t *>(table_out->pages);
    p.in_stride  = table->stride;
    p.out_stride = table_out->stride;
    p.n_seq      = table->n_seq;
    p.max_pages  = table->max_pages;
    p.len_in     = kv_len;
    p.len_out    = kv_len_out;
    p.refs_in    = refs;
    p.refs_out   = refs_out;
    p.src        = src;
    p.dst        = dst;
    p.n_pairs    = n_pairs;
    p.deep       = (flags & MM3FA_KV8_FORK_DEEP) != 0;
    return host_record_cuda(launch_kv8_fork(p, pool_copy(cache), host_sm_count(), static_cast<cudaStream_t>(stream)));
}

int mm3fa_kv8_compact(const mm3fa_kv8 * cache, const mm3fa_kv8_table * table, const int32_t * refs,
                      mm3fa_kv8_table * table_out, int32_t * refs_out, void * workspace, size_t workspace_bytes,
                      void * stream) {
    int           st = check_tables_out(cache, table, refs, table_out, refs_out);
    Kv8PlanParams p{};
    if (st == MM3FA_OK) {
        st = plan_workspace(cache, table, workspace, workspace_bytes, p);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    p.table_in   = table->pages;
    p.table_out  = const_cast<int32_t *>(table_out->pages);
    p.in_stride  = table->stride;
    p.out_stride = table_out->stride;
    p.n_seq      = table->n_seq;
    p.max_pages  = table->max_pages;
    p.refs_in    = refs;
    p.refs_out   = refs_out;
    return host_record_cuda(launch_kv8_compact(p, pool_copy(cache), host_sm_count(), static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
