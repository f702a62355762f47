// tree_abi.cu - C ABI of decoding with a tree of drafted tokens (the mm3fa_tree_* part of include/mm3fa.h).
//
// Checks the descriptors, fills the launch parameters and enqueues on the caller's stream; nothing allocates device
// memory or synchronises.
#include "../../include/mm3fa.h"
#include "tree.cuh"

#include <algorithm>
#include <cmath>
#include <cstdint>

using namespace mm3fa;

namespace {

bool aligned_to(const void * p, size_t a) {
    return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// Bytes of an element, or of a block of Q8_0 (0: no such type).
int64_t unit_bytes(int t) {
    return t == MM3FA_TYPE_F32 ? 4 : (t == MM3FA_TYPE_F16 || t == MM3FA_TYPE_BF16) ? 2 : t == MM3FA_TYPE_Q8_0 ? Q8_0_BLOCK : 0;
}

int64_t row_bytes(int t, int64_t n) {
    return t == MM3FA_TYPE_Q8_0 ? n / QK8_0 * Q8_0_BLOCK : n * unit_bytes(t);
}

int check_tree(const mm3fa_tree * t) {
    if (!t || !t->parents) {
        return MM3FA_ERR_NULL;
    }
    if (t->max_nodes < 1 || t->n_tree < 1 || t->stride < 0 || (t->n_tree > 1 && t->stride > 0 && t->stride < t->max_nodes)) {
        return MM3FA_ERR_SHAPE;
    }
    if (t->max_nodes > TREE_MAX || t->n_tree > 65535) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    return aligned_to(t->parents, 4) && aligned_to(t->n_nodes, 4) ? MM3FA_OK : MM3FA_ERR_ALIGN;
}

TreeDesc tree_of(const mm3fa_tree * t) {
    return { t->parents, t->stride, t->n_nodes, t->max_nodes, t->n_tree };
}

// A tensor whose rows are contiguous; the other strides are any multiples of an element (2 bytes for Q8_0).
int check_rows(const mm3fa_tensor * t, bool blocks) {
    if (!t) {
        return MM3FA_ERR_NULL;
    }
    const int64_t u = unit_bytes(t->type), a = t->type == MM3FA_TYPE_Q8_0 ? 2 : u;
    if (u == 0 || (!blocks && t->type == MM3FA_TYPE_Q8_0)) {
        return MM3FA_ERR_TYPE;
    }
    if (t->ne[0] < 1 || t->ne[1] < 1 || t->ne[2] < 1 || t->ne[3] < 1 || (t->type == MM3FA_TYPE_Q8_0 && t->ne[0] % QK8_0)) {
        return MM3FA_ERR_SHAPE;
    }
    if (!t->data) {
        return MM3FA_ERR_NULL;
    }
    if ((int64_t) t->nb[0] != u || t->nb[1] % a || t->nb[2] % a || t->nb[3] % a) {
        return MM3FA_ERR_STRIDE;
    }
    return aligned_to(t->data, (size_t) a) ? MM3FA_OK : MM3FA_ERR_ALIGN;
}

// Rows that are written: no two of them may share bytes through a stride below a row's.
bool rows_apart(const mm3fa_tensor * t) {
    for (int i = 1; i < 4; i++) {
        if (t->ne[i] > 1 && (int64_t) t->nb[i] < row_bytes(t->type, t->ne[0])) {
            return false;
        }
    }
    return true;
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

bool overlap(const void * a, size_t a_bytes, const void * b, size_t b_bytes) {
    const char * x = static_cast<const char *>(a), *y = static_cast<const char *>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

// Whether the K slab (V slab) of layer l is one that the list names before: layers that share their cache.  `apart`: none is.
bool named_before(const mm3fa_tensor * k, const mm3fa_tensor * v, int l, bool of_v, bool apart) {
    if (apart) {
        return false;
    }
    const void * x = of_v ? v[l].data : k[l].data;
    bool         alike = true;
    for (int i = 1; i < 4; i++) {
        alike = alike && (k->ne[i] == 1 || k->nb[i] == v->nb[i]);
    }
    for (int i = 0; i < l; i++) {
        if ((of_v ? v : k)[i].data == x || (alike && (of_v ? k : v)[i].data == x)) {
            return true;
        }
    }
    return of_v && alike && k[l].data == x;
}

// Whether all slabs are surely different ones: their addresses rise, K's apart from V's.
bool slabs_apart(const mm3fa_tensor * k, const mm3fa_tensor * v, int n) {
    for (int i = 1; i < n; i++) {
        if (k[i].data <= k[i - 1].data || v[i].data <= v[i - 1].data) {
            return false;
        }
    }
    return k[n - 1].data < v[0].data || v[n - 1].data < k[0].data;
}

// Whether a row of `a` and one of `b` share bytes, told from their extents, and, where these cross, for tensors whose strides
// are the same along each dimension (`of_b`: b's dimension of a's) and those above another's extent: rows in turn in one buffer.
// Others are taken to share some.
bool rows_share(const mm3fa_tensor * a, const mm3fa_tensor * b, const int (&of_b)[4]) {
    const int64_t wa = row_bytes(a->type, a->ne[0]), wb = row_bytes(b->type, b->ne[0]);
    int64_t       from_a = 0, end_a = wa, from_b = 0, end_b = wb;  // from the first row (strides may lead down)
    int           dims[3], n = 0;
    bool          alike = true;
    for (int i = 1; i < 4; i++) {
        const int     j = of_b[i];
        const int64_t ea = (a->ne[i] - 1) * (int64_t) a->nb[i], eb = (b->ne[j] - 1) * (int64_t) b->nb[j];
        (ea < 0 ? from_a : end_a) += ea, (eb < 0 ? from_b : end_b) += eb;
        if (a->ne[i] > 1) {
            alike     = alike && a->nb[i] == b->nb[j];
            dims[n++] = i;
        }
    }
    // a's first row from b's
    const int64_t d = (int64_t) (reinterpret_cast<uintptr_t>(a->data) - reinterpret_cast<uintptr_t>(b->data));
    if (d + from_a >= end_b || d + end_a <= from_b) {
        return false;
    }
    std::sort(dims, dims + n, [&](int x, int y) { return (int64_t) a->nb[x] > (int64_t) a->nb[y]; });
    int64_t below = std::max(wa, wb);  // of a row, or of the dimensions of smaller strides
    for (int k = n - 1; k >= 0; k--) {
        alike = alike && (int64_t) a->nb[dims[k]] >= below;
        below = (a->ne[dims[k]] - 1) * (int64_t) a->nb[dims[k]] + below;
    }
    if (!alike) {
        return true;
    }
    // Differences of two rows' places: d + sum of t_i nb_i, |t_i| < ne_i.  What the smaller strides add is less than a stride, so
    // that of each t_i two values can bring it near 0
    for (int pick = 0; pick < 1 << n; pick++) {
        int64_t x = d;
        for (int k = 0; k < n; k++) {
            const int64_t nb = (int64_t) a->nb[dims[k]], most = a->ne[dims[k]] - 1;
            const int64_t t  = -(x >= 0 ? x / nb : -((-x + nb - 1) / nb)) - (pick >> k & 1);
            x += std::min(std::max(t, -most), most) * nb;
        }
        if (x < wb && -x < wa) {
            return true;
        }
    }
    return false;
}

// The attention's operands; fills its parameters but for the workspace.
int prepare_attn(const mm3fa_tensor * q, const mm3fa_tensor * k, const mm3fa_tensor * v, const mm3fa_tree * tree, TreeAttnParams & p) {
    int st = check_tree(tree);
    if (st == MM3FA_OK) {
        st = check_rows(q, false);
    }
    for (const mm3fa_tensor * x : { k, v }) {
        if (st == MM3FA_OK) {
            st = check_rows(x, true);
        }
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (v->type != k->type) {
        return MM3FA_ERR_TYPE;
    }
    const int64_t D = q->ne[0], H = q->ne[2], S = q->ne[3];
    if (k->ne[0] != D || v->ne[0] != D || q->ne[1] != tree->max_nodes || v->ne[1] != k->ne[1] || v->ne[2] != k->ne[2] || k->ne[3] != S ||
        v->ne[3] != S || H % k->ne[2] || S % tree->n_tree) {
        return MM3FA_ERR_SHAPE;
    }
    if ((D != 64 && D != 128 && D != 256) || k->ne[1] > (1 << 30) || H > 16384 || H / k->ne[2] > 64 || S > 65535) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    p.t         = tree_of(tree);
    p.q         = rows_of(q);
    p.k         = rows_of(k);
    p.v         = rows_of(v);
    p.D         = (int) D;
    p.n_kv      = (int) k->ne[1];
    p.n_seq     = (int) S;
    p.n_head    = (int) H;
    p.n_head_kv = (int) k->ne[2];
    p.ratio     = (int) (H / k->ne[2]);
    return MM3FA_OK;
}

}  // namespace

extern "C" {

size_t mm3fa_tree_attn_workspace(const mm3fa_tensor * q, const mm3fa_tensor * k, const mm3fa_tensor * v, const mm3fa_tree * tree) {
    TreeAttnParams p{};
    // (the same for rows of every alignment and stride)
    return prepare_attn(q, k, v, tree, p) != MM3FA_OK ? 0 : tree_attn_tc_sizes(p) ? tree_attn_tc_workspace(p, host_sm_count()) : KV8_WS_ZEROED;
}

int mm3fa_tree_attn(const mm3fa_tensor * q, const mm3fa_tensor * k, const mm3fa_tensor * v, const mm3fa_tree * tree, const int32_t * kv_len,
                    float scale, float logit_softcap, mm3fa_tensor * dst, void * workspace, size_t workspace_bytes, void * stream) {
    TreeAttnParams p{};
    int            st = prepare_attn(q, k, v, tree, p);
    if (st == MM3FA_OK) {
        st = check_rows(dst, false);
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
    if (dst->ne[0] != q->ne[0] || dst->ne[1] != q->ne[2] || dst->ne[2] != q->ne[1] || dst->ne[3] != q->ne[3] || !std::isfinite(scale) ||
        !(logit_softcap >= 0.0f) || !std::isfinite(logit_softcap)) {
        return MM3FA_ERR_SHAPE;
    }
    if (!rows_apart(dst)) {
        return MM3FA_ERR_STRIDE;
    }
    if (!aligned_to(kv_len, 4)) {
        return MM3FA_ERR_ALIGN;
    }
    if (rows_share(q, dst, { 0, 2, 1, 3 })) {  // a CTA may still have to read what another writes
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < mm3fa_tree_attn_workspace(q, k, v, tree)) {
        return MM3FA_ERR_WORKSPACE;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    p.o          = rows_of(dst);
    p.kv_len     = kv_len;
    p.scale      = scale;
    // (from 1e30 on a cap changes no score of up to 1e26 in F32, and the quotients by it would leave F32's range)
    p.softcap    = logit_softcap < 1e30f ? logit_softcap : 0.0f;
    p.status     = static_cast<uint32_t *>(workspace);
    p.timeout_ns = host_wait_timeout_ns();
    // 16-bit slabs at D = 64 and 128 on the tensor cores; the others (F32, Q8_0, D = 256, unaligned rows) on CUDA cores
    return host_record_cuda(tree_attn_tc_takes(p) ? launch_tree_attn_tc(p, host_sm_count(), static_cast<cudaStream_t>(stream)) :
                                                    launch_tree_attn(p, static_cast<cudaStream_t>(stream)));
}

int mm3fa_tree_verify(const mm3fa_tensor * logits, const mm3fa_tensor * draft, const mm3fa_tree * tree, const int32_t * tokens,
                      const float * accept, const float * sample, float temperature, int32_t * path, int32_t * n_path, int32_t * token,
                      void * stream) {
    int st = check_tree(tree);
    if (st == MM3FA_OK) {
        st = check_rows(logits, false);
    }
    if (st == MM3FA_OK && draft) {
        st = check_rows(draft, false);
    }
    if (st != MM3FA_OK) {
        return st;
    }
    if (!tokens || !accept || !sample || !path || !n_path || !token) {
        return MM3FA_ERR_NULL;
    }
    for (const mm3fa_tensor * x : { logits, draft }) {
        if (x && (x->ne[0] != logits->ne[0] || x->ne[1] != tree->max_nodes || x->ne[2] != tree->n_tree || x->ne[3] != 1)) {
            return MM3FA_ERR_SHAPE;
        }
    }
    // the largest quotient of two logits' difference by the temperature stays a number
    const double inv_t = temperature == 0.0f ? 0.0 : 1.4426950408889634 / (double) temperature;
    if (!(temperature >= 0.0f) || !std::isfinite(temperature) || inv_t > 1e30) {
        return MM3FA_ERR_SHAPE;
    }
    if (logits->ne[0] > (1 << 22)) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    for (const void * x : { (const void *) tokens, (const void *) accept, (const void *) sample, (const void *) path, (const void *) n_path,
                            (const void *) token }) {
        if (!aligned_to(x, 4)) {
            return MM3FA_ERR_ALIGN;
        }
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    TreeVerifyParams p{};
    p.t      = tree_of(tree);
    p.logits = rows_of(logits);
    if (draft) {
        p.draft = rows_of(draft);
    }
    p.V      = (int) logits->ne[0];
    p.tokens = tokens;
    p.accept = accept;
    p.sample = sample;
    p.inv_t  = inv_t;
    p.path   = path;
    p.n_path = n_path;
    p.token  = token;
    return host_record_cuda(launch_tree_verify(p, host_sm_count(), static_cast<cudaStream_t>(stream)));
}

int mm3fa_tree_commit(const mm3fa_tensor * k, const mm3fa_tensor * v, int n_layers, const int32_t * path, const int32_t * n_path, int max_nodes,
                      int n_tree, const int32_t * kv_len, int32_t * kv_len_out, void * stream) {
    if (!k || !v || !path || !n_path || !kv_len || !kv_len_out) {
        return MM3FA_ERR_NULL;
    }
    if (n_layers < 1 || max_nodes < 1 || n_tree < 1) {
        return MM3FA_ERR_SHAPE;
    }
    if (max_nodes > TREE_MAX || n_tree > 65535) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    uintptr_t bits = 0;  // of all addresses and sizes
    for (int l = 0; l < n_layers; l++) {
        for (const mm3fa_tensor * x : { k + l, v + l }) {
            const int st = check_rows(x, true);
            if (st != MM3FA_OK) {
                return st;
            }
            const mm3fa_tensor * first = x == k + l ? k : v;
            if (x->type != k->type) {
                return MM3FA_ERR_TYPE;
            }
            for (int i = 0; i < 4; i++) {
                if (x->ne[i] != k->ne[i]) {
                    return MM3FA_ERR_SHAPE;
                }
                if (x->nb[i] != first->nb[i]) {
                    return MM3FA_ERR_STRIDE;
                }
            }
            if (!rows_apart(x)) {
                return MM3FA_ERR_STRIDE;
            }
            bits |= reinterpret_cast<uintptr_t>(x->data) | (x->ne[1] > 1 ? x->nb[1] : 0) | (x->ne[2] > 1 ? x->nb[2] : 0) | (x->ne[3] > 1 ? x->nb[3] : 0);
        }
    }
    const int64_t S = k->ne[3], row = row_bytes(k->type, k->ne[0]);
    if (S % n_tree) {
        return MM3FA_ERR_SHAPE;
    }
    // (sets and heads are counted in 32 bits)
    if (row > (1 << 20) || k->ne[2] > (1 << 20) || S > 65535 || 2 * (int64_t) TREE_LAYERS * S * k->ne[2] > INT32_MAX) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    for (const void * x : { (const void *) path, (const void *) n_path, (const void *) kv_len, (const void *) kv_len_out }) {
        if (!aligned_to(x, 4)) {
            return MM3FA_ERR_ALIGN;
        }
    }
    // every unit, and every launch of more than TREE_LAYERS layers, reads what one of them would replace
    const size_t out_bytes = 4 * (size_t) S, trees = (size_t) n_tree;
    if (overlap(kv_len, out_bytes, kv_len_out, out_bytes) || overlap(n_path, 4 * trees, kv_len_out, out_bytes) ||
        overlap(path, 4 * trees * (size_t) max_nodes, kv_len_out, out_bytes)) {
        return MM3FA_ERR_UNSUPPORTED;
    }
    if (host_device_major() != 10) {
        return MM3FA_ERR_DEVICE;
    }
    bits |= (uintptr_t) row;
    const int unit = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
    TreeCommitParams p{};
    p.k_nb1 = (int64_t) k->nb[1], p.k_nb2 = (int64_t) k->nb[2], p.k_nb3 = (int64_t) k->nb[3];
    p.v_nb1 = (int64_t) v->nb[1], p.v_nb2 = (int64_t) v->nb[2], p.v_nb3 = (int64_t) v->nb[3];
    p.row_bytes = (int) row;
    p.n_seq     = (int) S;
    p.n_head_kv = (int) k->ne[2];
    p.rows      = k->ne[1];
    p.path      = path;
    p.n_path    = n_path;
    p.kv_len    = kv_len;
    p.T         = max_nodes;
    p.n_tree    = n_tree;
    const bool apart = slabs_apart(k, v, n_layers);
    for (int l = 0; l < n_layers; l += TREE_LAYERS) {
        p.n_layers = std::min(TREE_LAYERS, n_layers - l);
        p.len_out  = l == 0 ? kv_len_out : nullptr;
        for (int i = 0; i < p.n_layers; i++) {
            p.k[i] = named_before(k, v, l + i, false, apart) ? nullptr : static_cast<char *>(k[l + i].data);
            p.v[i] = named_before(k, v, l + i, true, apart) ? nullptr : static_cast<char *>(v[l + i].data);
        }
        const int st = host_record_cuda(launch_tree_commit(p, unit, host_sm_count(), static_cast<cudaStream_t>(stream)));
        if (st != MM3FA_OK) {
            return st;
        }
    }
    return MM3FA_OK;
}

}  // extern "C"
