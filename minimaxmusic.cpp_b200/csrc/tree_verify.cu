// tree_verify.cu - which drafted tokens of a tree stay, and the token after them (sm_100a).
//
// The walk starts at node 0.  With p = softmax(logits of the current node / temperature) and q the distribution that its
// children were drawn from (the draft's, or 1 at a fixed choice), r = p and M = 1 at first, and for each child, in the
// order of the nodes, with token x and the given number u:
//     u q(x) M < r(x):  the child is accepted and becomes the current node
//     otherwise         r <- max(r - M q, 0),  M <- sum r
// What is left at the end gives the next token: the first x at which the sum of r up to it exceeds u' sum r.
// After k rejections r = max(p - c q, 0) with c the sum of the k values that M had, so that nothing but c is kept: no
// row of r is ever written.  With fixed choices r is p without the rejected tokens.
//
// One cluster of CTAs per tree, each with a slice of the vocabulary.  Only the rows of nodes on the path are read, one
// after another: T rows would be several times the bytes.  The sums over a row go from CTA to CTA through distributed
// shared memory, in the order of the ranks, and every thread takes the same decisions from them.
// The decisions come from F32 exponentials summed in F64; the last row's sums (and the M that lead to them) are taken in
// F64 throughout, since the next token's place among 10^5 borders moves with the twelfth digit of a partial sum.
#include "tree.cuh"

namespace mm3fa {

namespace {

constexpr int TV_THREADS = 1024;
constexpr int TV_WARPS   = TV_THREADS / 32;
constexpr int TV_CHUNK   = 256;  // entries whose sum is kept: 8 for each lane of a warp
constexpr int TV_E       = TV_CHUNK / 32;

struct TvShared {
    int    par[TREE_MAX], tok[TREE_MAX], path[TREE_MAX], gone[TREE_MAX];  // gone: rejected tokens (fixed choices)
    float  u[TREE_MAX], lx[TREE_MAX], qx[TREE_MAX];  // accept numbers; the token's logit and draft value in its parent's row
    double warp_a[TV_WARPS];
    float  warp_m[TV_WARPS];
    int    warp_i[TV_WARPS];
    double rank_a[2];  // what the other CTAs of the cluster read, in turn
    float  rank_m[2];
    int    rank_i[2];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t at_rank(const void * local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(local)), "r"(rank));
    return r;
}

__device__ __forceinline__ double ld_rank_f64(const double * local, uint32_t rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at_rank(local, rank)) : "memory");
    return v;
}

__device__ __forceinline__ float ld_rank_f32(const float * local, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at_rank(local, rank)) : "memory");
    return v;
}

__device__ __forceinline__ int ld_rank_i32(const int * local, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at_rank(local, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int TYPE>
__device__ __forceinline__ float load1(const char * row, int64_t i) {
    if (TYPE == KV_F32) {
        return reinterpret_cast<const float *>(row)[i];
    }
    if (TYPE == KV_F16) {
        return __half2float(reinterpret_cast<const __half *>(row)[i]);
    }
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(row)[i]);
}

// A logit as the sums take it: NaN counts as -inf, +inf as the largest number.
__device__ __forceinline__ float clean_logit(float x) {
    return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}

__device__ __forceinline__ float clean_draft(float q) {
    return fmaxf(q, 0.0f);  // NaN: 0
}

// LT, DT: types of logits and drafts (DT -1: fixed choices)
template <int LT, int DT>
struct Walk {
    const TreeVerifyParams & p;
    TvShared &               sh;
    double *                 sums;  // of the CTA's chunks
    const char *             lrow;  // the current node's rows
    const char *             qrow;
    int                      lo, hi, n_ranks;  // the CTA's slice
    uint32_t                 rank;
    int                      turn;
    int                      tid, lane, warp;

    __device__ __forceinline__ void sync() const {
        if (n_ranks > 1) {
            cluster_sync();
        } else {
            __syncthreads();
        }
    }

    // the sum of a value of every thread over the cluster, the same in every thread
    __device__ double total(double a) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
        }
        __syncthreads();  // (what the call before read has been read)
        if (lane == 0) {
            sh.warp_a[warp] = a;
        }
        __syncthreads();
        a = 0.0;
#pragma unroll 8
        for (int w = 0; w < TV_WARPS; w++) {
            a += sh.warp_a[w];
        }
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_a[turn] = a;
            }
            cluster_sync();
            a = 0.0;
            for (int r = 0; r < n_ranks; r++) {
                a += ld_rank_f64(&sh.rank_a[turn], r);
            }
            turn ^= 1;
        }
        return a;
    }

    // (m, sum of 2^((x - m) / t)) over the row
    __device__ void row_mass(float & m_out, double & z_out) {
        const float a = (float) p.inv_t;
        float       m = -INFINITY, s = 0.0f;
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += TV_WARPS * TV_CHUNK) {
            float x[TV_E], top = -INFINITY;
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                const int i = i0 + e * 32 + lane;
                x[e]        = i < hi ? clean_logit(load1<LT>(lrow, i)) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                top = fmaxf(top, x[e]);
            }
            if (top > m) {
                s *= exp2f((m - top) * a);
                m = top;
            }
            if (m > -INFINITY) {
#pragma unroll
                for (int e = 0; e < TV_E; e++) {
                    s += exp2f((x[e] - m) * a);
                }
            }
        }
        float top = m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        }
        double z = m > -INFINITY ? (double) s * (double) exp2f((m - top) * a) : 0.0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, d);
        }
        __syncthreads();
        if (lane == 0) {
            sh.warp_m[warp] = top, sh.warp_a[warp] = z;
        }
        __syncthreads();
        m = -INFINITY;
#pragma unroll 8
        for (int w = 0; w < TV_WARPS; w++) {
            m = fmaxf(m, sh.warp_m[w]);
        }
        z = 0.0;
#pragma unroll 8
        for (int w = 0; w < TV_WARPS; w++) {
            z += sh.warp_m[w] > -INFINITY ? sh.warp_a[w] * (double) exp2f((sh.warp_m[w] - m) * a) : 0.0;
        }
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_m[turn] = m, sh.rank_a[turn] = z;
            }
            cluster_sync();
            m = -INFINITY;
            for (int r = 0; r < n_ranks; r++) {
                m = fmaxf(m, ld_rank_f32(&sh.rank_m[turn], r));
            }
            z = 0.0;
            for (int r = 0; r < n_ranks; r++) {
                const float mr = ld_rank_f32(&sh.rank_m[turn], r);
                z += mr > -INFINITY ? ld_rank_f64(&sh.rank_a[turn], r) * (double) exp2f((mr - m) * a) : 0.0;
            }
            turn ^= 1;
        }
        m_out = m, z_out = z;
    }

    // the lowest index of the row's largest logit (-1: none is above -inf)
    __device__ int row_argmax() {
        float m = -INFINITY;
        int   at = 0x7fffffff;
        for (int i = lo + tid; i < hi; i += TV_THREADS) {
            const float x = clean_logit(load1<LT>(lrow, i));
            if (x > m) {
                m = x, at = i;
            }
        }
        auto take = [&](float x, int i) {
            if (x > m || (x == m && i < at)) {
                m = x, at = i;
            }
        };
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const float x = __shfl_xor_sync(0xffffffffu, m, d);
            take(x, __shfl_xor_sync(0xffffffffu, at, d));
        }
        __syncthreads();
        if (lane == 0) {
            sh.warp_m[warp] = m, sh.warp_i[warp] = at;
        }
        __syncthreads();
        for (int w = 0; w < TV_WARPS; w++) {
            take(sh.warp_m[w], sh.warp_i[w]);
        }
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_m[turn] = m, sh.rank_i[turn] = at;
            }
            cluster_sync();
            for (int r = 0; r < n_ranks; r++) {
                take(ld_rank_f32(&sh.rank_m[turn], r), ld_rank_i32(&sh.rank_i[turn], r));
            }
            turn ^= 1;
        }
        return m > -INFINITY ? at : -1;
    }

    // sum of max(p - c q, 0), in F32 terms
    __device__ double left_mass(float m, double z, double c) {
        const float a = (float) p.inv_t, iz = (float) (1.0 / z), cf = (float) c;
        double      sum = 0.0;
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += TV_WARPS * TV_CHUNK) {
            float x[TV_E], q[TV_E], s = 0.0f;
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                const int i = i0 + e * 32 + lane;
                x[e]        = i < hi ? clean_logit(load1<LT>(lrow, i)) : -INFINITY;
                q[e]        = i < hi ? clean_draft(load1<DT>(qrow, i)) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                s += fmaxf(exp2f((x[e] - m) * a) * iz - cf * q[e], 0.0f);
            }
            sum += (double) s;
        }
        return total(sum);
    }

    __device__ __forceinline__ double weight(float x, float m) const {
        return exp2(((double) x - (double) m) * p.inv_t);
    }

    // what is left of entry i: max(p - c q, 0), or the weight of a token that was not rejected
    __device__ __forceinline__ double left(int i, float m, double iz, double c, int n_gone) const {
        double w = weight(clean_logit(load1<LT>(lrow, i)), m);
        if constexpr (DT >= 0) {
            return c > 0.0 ? fmax(w * iz - c * (double) clean_draft(load1<DT>(qrow, i)), 0.0) : w;
        } else {
            for (int k = 0; k < n_gone; k++) {
                w = sh.gone[k] == i ? 0.0 : w;
            }
            return w;
        }
    }

    // sum of `left` over the row; the sums of the CTA's chunks are kept
    __device__ double left_sums(float m, double iz, double c, int n_gone) {
        double sum = 0.0;
        __syncthreads();
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += TV_WARPS * TV_CHUNK) {
            double s = 0.0;
#pragma unroll 4
            for (int e = 0; e < TV_E; e++) {
                const int i = i0 + e * 32 + lane;
                s += i < hi ? left(i, m, iz, c, n_gone) : 0.0;
            }
            sum += s;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, d);
            }
            if (lane == 0) {
                sums[(i0 - lo) / TV_CHUNK] = s;
            }
        }
        return total(sum);
    }

    // the first entry at which the sum of what is left exceeds u times all of it, by the CTA that holds it; the chunks'
    // sums of the last left_sums() are in place
    __device__ void sample(float u, float m, double iz, double c, int n_gone, int * out) {
        const int n_chunks = hi > lo ? (hi - lo + TV_CHUNK - 1) / TV_CHUNK : 0;
        // this CTA's sum, and the ranks' before it, from the same numbers in the same order everywhere
        __syncthreads();
        double mine = 0.0;
        if (warp == 0) {
            for (int k = lane; k < n_chunks; k += 32) {
                mine += sums[k];
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                mine += __shfl_xor_sync(0xffffffffu, mine, d);
            }
        }
        if (tid == 0) {
            sh.rank_a[turn] = mine;
        }
        sync();
        if (warp == 0) {
            double all = 0.0, before = 0.0;
            int    last = -1, owner = -1;
            for (int r = 0; r < n_ranks; r++) {
                all += ld_rank_f64(&sh.rank_a[turn], r);
            }
            const double target = (double) fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f) * all;
            double       run = 0.0;
            for (int r = 0; r < n_ranks; r++) {
                const double x = ld_rank_f64(&sh.rank_a[turn], r);
                if (x > 0.0) {
                    last = r;
                    if (owner < 0 && run + x > target) {
                        owner = r, before = run;
                    }
                }
                run += x;
            }
            if (owner < 0) {  // (cannot be: the sums of ranks end at `all`, which is above the target)
                owner = last, before = -INFINITY;
            }
            if (owner == (int) rank) {
                // the chunk, then the entry: a warp's prefix sums over the rest that is in the way
                int    chunk = -1;
                double start = before;
                for (int k0 = 0; k0 < n_chunks && chunk < 0; k0 += 32) {
                    const double x = k0 + lane < n_chunks ? sums[k0 + lane] : 0.0;
                    double       s = x;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, s, d);
                        s += lane >= d ? y : 0.0;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, x > 0.0 && start + s > target);
                    if (over) {
                        const int k = __ffs(over) - 1;
                        chunk       = k0 + k;
                        start += __shfl_sync(0xffffffffu, s - x, k);
                    } else {
                        start += __shfl_sync(0xffffffffu, s, 31);
                    }
                }
                if (chunk < 0) {  // roundings between two orders of summing: the last entry that holds anything
                    for (int k = 0; k < n_chunks; k++) {
                        chunk = sums[k] > 0.0 ? k : chunk;
                    }
                    start = -INFINITY;
                }
                int token = -1, backup = -1;
                for (int e = 0; e < TV_E && token < 0; e++) {
                    const int    i = lo + chunk * TV_CHUNK + e * 32 + lane;
                    const double x = i < hi ? left(i, m, iz, c, n_gone) : 0.0;
                    double       s = x;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const double y = __shfl_up_sync(0xffffffffu, s, d);
                        s += lane >= d ? y : 0.0;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, x > 0.0 && start + s > target);
                    const unsigned some = __ballot_sync(0xffffffffu, x > 0.0);
                    if (over) {
                        token = lo + chunk * TV_CHUNK + e * 32 + __ffs(over) - 1;
                    }
                    backup = some ? lo + chunk * TV_CHUNK + e * 32 + 31 - __clz(some) : backup;
                    start += __shfl_sync(0xffffffffu, s, 31);
                }
                if (lane == 0) {
                    *out = token >= 0 ? token : backup;
                }
            }
        }
        turn ^= 1;
    }
};

template <int LT, int DT>
__global__ void __launch_bounds__(TV_THREADS, 1) tree_verify_kernel(const TreeVerifyParams p, int n_ranks) {
    kv8_dep_wait();
    extern __shared__ double tv_sums[];
    __shared__ TvShared      sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = p.t.max_nodes;
    const int tree = (int) blockIdx.x / n_ranks;
    const uint32_t rank = n_ranks > 1 ? cluster_rank() : 0;
    const int n    = tree_nodes(p.t, tree);
    int * path     = p.path + (int64_t) tree * T;
    if (n == 0) {
        if (rank == 0) {
            for (int i = tid; i < T; i += TV_THREADS) {
                path[i] = -1;
            }
            if (tid == 0) {
                p.n_path[tree] = 0, p.token[tree] = -1;
            }
        }
        return;
    }
    const char * lbase = p.logits.data + (int64_t) tree * p.logits.nb2, *qbase = DT >= 0 ? p.draft.data + (int64_t) tree * p.draft.nb2 : nullptr;
    for (int i = tid; i < n; i += TV_THREADS) {
        const int pr = tree_parent(p.t, tree, i), x = p.tokens[(int64_t) tree * T + i];
        const bool ok = i > 0 && pr >= 0 && x >= 0 && x < p.V;  // a token outside the vocabulary is never accepted
        sh.par[i] = ok ? pr : -1, sh.tok[i] = x, sh.u[i] = p.accept[(int64_t) tree * T + i];
        sh.lx[i] = ok ? clean_logit(load1<LT>(lbase + (int64_t) pr * p.logits.nb1, x)) : -INFINITY;
        sh.qx[i] = 1.0f;
        if (DT >= 0) {
            sh.qx[i] = ok ? clean_draft(load1<DT>(qbase + (int64_t) pr * p.draft.nb1, x)) : 0.0f;
        }
    }
    // slices of whole chunks
    const int chunks = (p.V + TV_CHUNK - 1) / TV_CHUNK, each = (chunks + n_ranks - 1) / n_ranks;
    Walk<LT, DT> w{ p, sh, tv_sums, lbase, qbase, 0, 0, n_ranks, rank, 0, tid, lane, warp };
    w.lo = min((int) rank * each * TV_CHUNK, p.V), w.hi = min(((int) rank + 1) * each * TV_CHUNK, p.V);
    __syncthreads();
    int    cur = 0, n_path = 1, n_gone, n_no, best = -1;
    float  m = 0.0f;
    double z = 0.0;
    if (tid == 0) {
        sh.path[0] = 0;
    }
    for (;;) {
        w.lrow = lbase + (int64_t) cur * p.logits.nb1;
        w.qrow = DT >= 0 ? qbase + (int64_t) cur * p.draft.nb1 : nullptr;
        n_gone = n_no = 0;
        const bool greedy = p.inv_t == 0.0;
        if (greedy) {
            best = w.row_argmax();
        } else {
            w.row_mass(m, z);
            best = m > -INFINITY ? 0 : -1;
        }
        int    next = -1;
        double c = 0.0, M = 1.0;
        for (int k0 = cur / 32 * 32; best >= 0 && next < 0 && k0 < n; k0 += 32) {
            unsigned kids = __ballot_sync(0xffffffffu, k0 + lane < n && k0 + lane > cur && sh.par[min(k0 + lane, TREE_MAX - 1)] == cur);
            while (kids && next < 0) {
                const int i = k0 + __ffs(kids) - 1;
                kids &= kids - 1;
                if (greedy) {
                    next = sh.tok[i] == best ? i : -1;
                    continue;
                }
                const double px = w.weight(sh.lx[i], m) / z, q = (double) sh.qx[i];
                double       r  = fmax(px - c * q, 0.0);
                if (DT < 0) {
                    r = px;
                    for (int k = 0; k < n_gone; k++) {
                        r = sh.gone[k] == sh.tok[i] ? 0.0 : r;
                    }
                }
                if ((double) sh.u[i] * q * M < r) {
                    next = i;
                } else if (DT >= 0) {
                    c += M;
                    n_no++;
                    M = w.left_mass(m, z, c);
                } else if (r > 0.0) {
                    M = fmax(M - r, 0.0);
                    __syncthreads();
                    if (tid == 0) {
                        sh.gone[n_gone] = sh.tok[i];
                    }
                    __syncthreads();
                    n_gone++;
                }
            }
        }
        if (next < 0) {
            break;
        }
        cur = next;
        if (tid == 0) {
            sh.path[n_path] = cur;
        }
        n_path++;
    }
    if (p.inv_t != 0.0 && best >= 0) {
        double iz = 1.0, c = 0.0;
        if (DT >= 0 && n_no > 0) {
            iz = 1.0 / w.left_sums(m, 1.0, 0.0, 0);
            c  = 1.0;
            for (int k = 1; k < n_no; k++) {
                c += w.left_sums(m, iz, c, 0);
            }
        }
        if (!(w.left_sums(m, iz, c, n_gone) > 0.0)) {  // nothing is left: the target's own distribution
            c = 0.0, n_gone = 0;
            w.left_sums(m, iz, c, n_gone);
        }
        w.sample(p.sample[tree], m, iz, c, n_gone, p.token + tree);
    } else if (rank == 0 && tid == 0) {
        p.token[tree] = best;
    }
    __syncthreads();
    if (rank == 0) {
        for (int i = tid; i < T; i += TV_THREADS) {
            path[i] = i < n_path ? sh.path[i] : -1;
        }
        if (tid == 0) {
            p.n_path[tree] = n_path;
        }
    }
    if (n_ranks > 1) {
        cluster_sync();  // a CTA's shared memory stays until the others have read it
    }
}

template <int LT, int DT>
cudaError_t launch_one(const TreeVerifyParams & p, int n_ranks, cudaStream_t stream) {
    static Kv8Once once;
    const int      chunks = (p.V + TV_CHUNK - 1) / TV_CHUNK;
    const size_t   smem   = (size_t) ((chunks + n_ranks - 1) / n_ranks) * sizeof(double);
    cudaError_t    e      = once.smem(tree_verify_kernel<LT, DT>, 160 << 10);
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim          = dim3((unsigned) (p.t.n_tree * n_ranks));
    cfg.blockDim         = dim3(TV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream           = stream;
    cfg.attrs            = attr;
    cfg.numAttrs         = 0;
    if (n_ranks > 1) {
        attr[cfg.numAttrs].id               = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = (unsigned) n_ranks;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    if (kv8_pdl()) {
        attr[cfg.numAttrs].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs++;
    }
    return cudaLaunchKernelEx(&cfg, tree_verify_kernel<LT, DT>, p, n_ranks);
}

template <int LT>
cudaError_t launch_l(const TreeVerifyParams & p, int n_ranks, cudaStream_t stream) {
    if (!p.draft.data) {
        return launch_one<LT, -1>(p, n_ranks, stream);
    }
    switch (p.draft.type) {
        case KV_F32:
            return launch_one<LT, KV_F32>(p, n_ranks, stream);
        case KV_F16:
            return launch_one<LT, KV_F16>(p, n_ranks, stream);
        default:
            return launch_one<LT, KV_BF16>(p, n_ranks, stream);
    }
}

}  // namespace

cudaError_t launch_tree_verify(const TreeVerifyParams & p, int sms, cudaStream_t stream) {
    // CTAs of a tree: as many as the SMs give each tree, up to 8 (the portable size), with two chunks a warp or more
    int n_ranks = 1;
    while (n_ranks < 8 && 2 * n_ranks * p.t.n_tree <= sms && p.V >= 2 * n_ranks * TV_WARPS * TV_CHUNK / 4) {
        n_ranks *= 2;
    }
    switch (p.logits.type) {
        case KV_F32:
            return launch_l<KV_F32>(p, n_ranks, stream);
        case KV_F16:
            return launch_l<KV_F16>(p, n_ranks, stream);
        default:
            return launch_l<KV_BF16>(p, n_ranks, stream);
    }
}

}  // namespace mm3fa
