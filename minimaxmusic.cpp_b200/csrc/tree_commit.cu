// tree_commit.cu - the cache rows of a tree's accepted nodes moved behind the tokens that a sequence holds (sm_100a).
//
// Row L + path[i] goes to row L + i, for K and V of every layer, set and kv head.  One warp per (layer, K or V, set,
// head): it holds TC_ROWS rows at a time in registers, loads before stores.  The path rises and path[i] >= i, so a row
// written for one batch of rows is never a source of a later one, and the move can be done in place.
// Bound: HBM for large batches, launch and two dependent reads (path, then rows) for small ones.
#include "tree.cuh"

namespace mm3fa {

namespace {

constexpr int TC_WARPS = 8;

template <typename U>
__global__ void __launch_bounds__(32 * TC_WARPS) tree_commit_kernel(const __grid_constant__ TreeCommitParams p) {
    kv8_dep_wait();
    const int     lane = threadIdx.x & 31;
    const int64_t unit = (int64_t) blockIdx.x * TC_WARPS + (threadIdx.x >> 5), heads = (int64_t) p.n_seq * p.n_head_kv;
    if (unit >= 2 * p.n_layers * heads) {
        return;
    }
    const int layer = (int) (unit / (2 * heads)), which = (int) (unit / heads & 1), s = (int) (unit % heads / p.n_head_kv), h = (int) (unit % p.n_head_kv);
    const int tree = s % p.n_tree, held = p.kv_len[s];
    const int * path = p.path + (int64_t) tree * p.T;
    const int   most = min(max(p.n_path[tree], 0), p.T);
    char *      base = which ? p.v[layer] + (int64_t) h * p.v_nb2 + (int64_t) s * p.v_nb3 : p.k[layer] + (int64_t) h * p.k_nb2 + (int64_t) s * p.k_nb3;
    const int64_t nb1 = which ? p.v_nb1 : p.k_nb1;
    const int pieces = p.row_bytes / (int) sizeof(U);
    int       n = 0, before = -1;
    for (int i0 = 0; i0 < most; i0 += 32) {
        // the path ends at an entry that does not rise or names no row of the slab
        const int      at = i0 + lane < most ? path[i0 + lane] : -1;
        int            prev = __shfl_up_sync(0xffffffffu, at, 1);
        prev                = lane == 0 ? before : prev;
        const bool     ok   = i0 + lane < most && held >= 0 && at > prev && at < p.T && (int64_t) held + at < p.rows;
        const unsigned good = __ballot_sync(0xffffffffu, ok);
        const int      rows = good == 0xffffffffu ? 32 : __ffs(~good) - 1;
        before              = __shfl_sync(0xffffffffu, at, 31);
        // rows that are where they belong already are left out: the first ones
        const unsigned stay = __ballot_sync(0xffffffffu, at == i0 + lane);
        const int      skip = stay == 0xffffffffu ? 32 : __ffs(~stay) - 1;
        constexpr int  B    = 4;
        const int      items = rows * pieces;
        for (int e0 = min(skip, rows) * pieces; e0 < items; e0 += 32 * B) {
            // (whole batches of rows would do; batches of pieces do as well: a later batch's sources lie at or
            // behind its own destinations, which lie behind those of this batch)
            U x[B];
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int e = e0 + b * 32 + lane, r = min(e / pieces, 31), src = __shfl_sync(0xffffffffu, at, r);
                if (e < items) {
                    x[b] = *reinterpret_cast<const U *>(base + ((int64_t) held + src) * nb1 + (e - r * pieces) * (int) sizeof(U));
                }
            }
            __syncwarp();
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int e = e0 + b * 32 + lane, r = e / pieces;
                if (e < items) {
                    *reinterpret_cast<U *>(base + ((int64_t) held + i0 + r) * nb1 + (e - r * pieces) * (int) sizeof(U)) = x[b];
                }
            }
            __syncwarp();
        }
        n += rows;
        if (rows < 32) {
            break;
        }
    }
    if (p.len_out && layer == 0 && which == 0 && h == 0 && lane == 0) {
        p.len_out[s] = held + n;
    }
}

template <typename U>
cudaError_t launch_one(const TreeCommitParams & p, cudaStream_t stream) {
    const int64_t units = (int64_t) 2 * p.n_layers * p.n_seq * p.n_head_kv;
    return kv8_launch(tree_commit_kernel<U>, dim3((unsigned) ((units + TC_WARPS - 1) / TC_WARPS)), 32 * TC_WARPS, 0, stream, p);
}

}  // namespace

// unit: the widest access, in bytes, that every row's address and size allow
cudaError_t launch_tree_commit(const TreeCommitParams & p, int unit, cudaStream_t stream) {
    switch (unit) {
        case 16:
            return launch_one<uint4>(p, stream);
        case 8:
            return launch_one<uint2>(p, stream);
        case 4:
            return launch_one<uint32_t>(p, stream);
        default:
            return launch_one<uint16_t>(p, stream);
    }
}

}  // namespace mm3fa
