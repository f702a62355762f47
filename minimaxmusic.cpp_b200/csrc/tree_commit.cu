// tree_commit.cu - the cache rows of a tree's accepted nodes moved behind the tokens that a sequence holds (sm_100a).
//
// Row L + path[i] goes to row L + i, for K and V of every layer, set and kv head.  A warp has K and V of a set and head, in one
// layer or in several where there are warps enough: the path is read once, and a batch's pieces of rows are all loaded, of
// both, before the first is stored.  The path rises and path[i] >= i, so a row written is never a source of a later
// batch, and the move can be done in place.
// Bound: HBM for large batches, launch and two dependent reads (path, then rows) for small ones.  36 layers, 48 sets, 8
// heads, 3.4 rows of 256 bytes a head (47.8 MB read and written): 8.8 us from HBM, 6.2 us where L2 holds the rows; one
// layer of K or V a warp, with places by 64-bit divisions: 17.6 and 15.2 us.  36 layers of 2 sets: 2.1 us.
#include "tree.cuh"

#include <algorithm>

namespace mm3fa {

namespace {

constexpr int TC_WARPS = 8;

template <typename U>
__global__ void __launch_bounds__(32 * TC_WARPS) tree_commit_kernel(const __grid_constant__ TreeCommitParams p) {
    kv8_dep_wait();
    const int lane = threadIdx.x & 31, unit = (int) blockIdx.x * TC_WARPS + (int) threadIdx.x / 32;
    if (unit >= p.n_seq * p.n_head_kv) {
        return;
    }
    const int     s = unit / p.n_head_kv, h = unit - s * p.n_head_kv, tree = s % p.n_tree, held = p.kv_len[s];
    const int *   path = p.path + (int64_t) tree * p.T;
    const int     most = min(max(p.n_path[tree], 0), p.T), pieces = p.row_bytes / (int) sizeof(U);
    const int64_t k0 = (int64_t) h * p.k_nb2 + (int64_t) s * p.k_nb3 + (int64_t) held * p.k_nb1;
    const int64_t v0 = (int64_t) h * p.v_nb2 + (int64_t) s * p.v_nb3 + (int64_t) held * p.v_nb1;
    int           n = 0, before = -1;
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
        const int      skip = stay == 0xffffffffu ? 32 : __ffs(~stay) - 1, items = rows * pieces;
        constexpr int  B    = 4;
        for (int layer = blockIdx.y; layer < p.n_layers; layer += (int) gridDim.y) {
            const bool has_k = p.k[layer] != nullptr, has_v = p.v[layer] != nullptr;
            char * k = p.k[layer] + k0, *v = p.v[layer] + v0;
            for (int e0 = min(skip, rows) * pieces; e0 < items; e0 += 32 * B) {
                // (batches may end inside a row: a later batch's sources lie at or behind its own destinations, which lie
                // behind those of this batch)
                U x[B], y[B];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const int e = e0 + b * 32 + lane, r = min(e / pieces, 31), src = __shfl_sync(0xffffffffu, at, r);
                    if (e < items) {
                        const int64_t off = (int64_t) (e - r * pieces) * (int) sizeof(U);
                        if (has_k) {
                            x[b] = *reinterpret_cast<const U *>(k + src * p.k_nb1 + off);
                        }
                        if (has_v) {
                            y[b] = *reinterpret_cast<const U *>(v + src * p.v_nb1 + off);
                        }
                    }
                }
                __syncwarp();
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const int e = e0 + b * 32 + lane, r = e / pieces;
                    if (e < items) {
                        const int64_t off = (int64_t) (e - r * pieces) * (int) sizeof(U);
                        if (has_k) {
                            *reinterpret_cast<U *>(k + (i0 + r) * p.k_nb1 + off) = x[b];
                        }
                        if (has_v) {
                            *reinterpret_cast<U *>(v + (i0 + r) * p.v_nb1 + off) = y[b];
                        }
                    }
                }
                __syncwarp();
            }
        }
        n += rows;
        if (rows < 32) {
            break;
        }
    }
    if (p.len_out && blockIdx.y == 0 && h == 0 && lane == 0) {
        p.len_out[s] = held + n;
    }
}

template <typename U>
cudaError_t launch_one(const TreeCommitParams & p, int sms, cudaStream_t stream) {
    // layers of a warp: one, until that is more than 32 warps an SM
    const int64_t heads = (int64_t) p.n_seq * p.n_head_kv;
    const int     each  = (int) std::max<int64_t>(1, std::min<int64_t>(p.n_layers, heads * p.n_layers / (32 * (int64_t) std::max(sms, 1))));
    return kv8_launch(tree_commit_kernel<U>, dim3((unsigned) ((heads + TC_WARPS - 1) / TC_WARPS), (unsigned) ((p.n_layers + each - 1) / each)), 32 * TC_WARPS, 0,
                      stream, p);
}

}  // namespace

// unit: the widest access, in bytes, that every row's address and size allow
cudaError_t launch_tree_commit(const TreeCommitParams & p, int unit, int sms, cudaStream_t stream) {
    switch (unit) {
        case 16:
            return launch_one<uint4>(p, sms, stream);
        case 8:
            return launch_one<uint2>(p, sms, stream);
        case 4:
            return launch_one<uint32_t>(p, sms, stream);
        default:
            return launch_one<uint16_t>(p, sms, stream);
    }
}

}  // namespace mm3fa
