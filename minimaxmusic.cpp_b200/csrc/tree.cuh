// tree.cuh - decoding with a tree of drafted tokens: launch parameters and helpers shared by its kernels (sm_100a).
//
// A tree has up to TREE_MAX nodes; parents[i] < i names a node's parent (anything else: none).  Sequence s goes by
// tree s % n_tree.  The K and V rows of node i of a sequence that holds L tokens are rows L + i of its cache slab.
#pragma once

#include "kv8.cuh"

namespace mm3fa {

constexpr int TREE_MAX    = 256;  // nodes of a tree, at most
constexpr int TREE_LAYERS = 96;   // layers of one launch of the commit, at most (their addresses are kernel parameters)

struct TreeDesc {
    const int * parents;  // [n_tree][stride]
    int64_t     stride;   // entries
    const int * n_nodes;  // [n_tree] or null: max_nodes
    int         max_nodes, n_tree;
};

struct TreeAttnParams {
    TreeDesc    t;
    Kv8Rows     q, o;    // q [D, T, H, S]; o [D, H, T, S]
    Kv8Rows     k, v;    // [D, n_kv, Hkv, S]
    const int * kv_len;  // [S]
    int         D, n_kv, n_seq, n_head, n_head_kv, ratio;
    float       scale, softcap;
    // workspace
    uint32_t *  status;
    float *     part;
    uint64_t    timeout_ns;
};

struct TreeVerifyParams {
    TreeDesc      t;
    Kv8Rows       logits, draft;  // [V, T, n_tree]; draft.data null: the drafts are fixed choices
    int           V;
    const int *   tokens;  // [n_tree][T]
    const float * accept;  // [n_tree][T]
    const float * sample;  // [n_tree]
    double        inv_t;   // log2(e) / temperature; 0: greedy
    int *         path;    // [n_tree][T]
    int *         n_path;  // [n_tree]
    int *         token;   // [n_tree]
};

struct TreeCommitParams {
    char *      k[TREE_LAYERS];  // null: a slab that was named before, which is moved once
    char *      v[TREE_LAYERS];
    int64_t     k_nb1, k_nb2, k_nb3, v_nb1, v_nb2, v_nb3;
    int         row_bytes;
    int         n_layers, n_seq, n_head_kv;
    int64_t     rows;    // of a slab
    const int * path;    // [n_tree][T]
    const int * n_path;  // [n_tree]
    const int * kv_len;  // [S]
    int *       len_out; // [S]; null: a later launch of the same call writes it
    int         T, n_tree;
};

__device__ __forceinline__ int tree_nodes(const TreeDesc & t, int tree) {
    return t.n_nodes ? min(max(t.n_nodes[tree], 0), t.max_nodes) : t.max_nodes;
}

// A node's parent, -1 where it has none.
__device__ __forceinline__ int tree_parent(const TreeDesc & t, int tree, int i) {
    const int p = t.parents[(int64_t) tree * t.stride + i];
    return p >= 0 && p < i ? p : -1;
}

cudaError_t launch_tree_attn(const TreeAttnParams & p, cudaStream_t stream);
bool        tree_attn_tc_takes(const TreeAttnParams & p);
bool        tree_attn_tc_sizes(const TreeAttnParams & p);  // the same, but for the alignment and strides of rows
int         tree_attn_wide(const TreeAttnParams & p);  // CTAs of a group
int         tree_attn_groups(const TreeAttnParams & p, int keys, int sms);
size_t      tree_attn_tc_workspace(const TreeAttnParams & p, int sms);
cudaError_t launch_tree_attn_tc(TreeAttnParams p, int sms, cudaStream_t stream);
cudaError_t launch_tree_verify(const TreeVerifyParams & p, int sms, cudaStream_t stream);
cudaError_t launch_tree_commit(const TreeCommitParams & p, int unit, int sms, cudaStream_t stream);

}  // namespace mm3fa
