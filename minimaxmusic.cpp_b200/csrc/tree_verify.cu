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
// A decision is what F64 sums say, to 12 digits.  A row's first sum, and the M of drafts, are of F32 exponentials and off by
// TV_CLOSE at most; where a decision is nearer to its border than that, and for the next token, whose place among 10^5 borders
// moves with the twelfth digit of a partial sum, the row is summed again in F64 (and what the fixed choices that were turned
// down leave is summed without them, so that a child with nearly all of the probability leaves all its digits to the rest).
//
// Bound: HBM where there are many trees, else the passes of a walk, one after another (a row, and a rejection's sum): a slice
// of up to 8 entries a thread is kept in registers between them.  F64 runs at half of F32's rate here, and exp2() is some
// 40 instructions of it: with a table of 32 powers, one in each lane, and a polynomial it is 8.
#include "tree.cuh"

#include <type_traits>

namespace mm3fa {

namespace {

constexpr int TV_THREADS = 1024;  // of a CTA, at most
constexpr int TV_WARPS   = TV_THREADS / 32;
constexpr int TV_RANKS   = 8;     // CTAs of a tree, at most
constexpr int TV_CHUNK   = 256;   // entries whose sum is kept: 8 for each lane of a warp
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

// 2^y on the special-function unit, 0 below 2^-126
__device__ __forceinline__ float power2(float y) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}

// A logit as the sums take it: NaN counts as -inf, +inf as the largest number.
__device__ __forceinline__ float clean_logit(float x) {
    return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);  // (the maximum of NaN and a number is the number)
}

__device__ __forceinline__ float clean_draft(float q) {
    return fmaxf(q, 0.0f);  // NaN: 0
}

// sum + 2^(d t) for exponents from -1000 to 0, to 12 digits: the exponent is n + k / 32 + r with |r| <= 1/64; 2^(k / 32) comes
// from lane k (`power` of each lane), n goes into its exponent, and 2^r is its series to the fourth power.  `none`: sum, and
// less than 2^-1000.  By whole warps; 8 instructions of F64.
__device__ __forceinline__ double add_power(double d, double t, double power, bool none, double sum) {
    const double magic = 0x1.8p+47;  // a number this large is a multiple of 1/32
    const double y = fma(d, t, magic), r = fma(d, t, magic - y);
    const int    n = __double2loint(y);  // 32 n + k
    const double pw = __shfl_sync(0xffffffffu, power, n & 31);
    // ln(2)^i / i!
    double s = fma(9.618129107628477e-3, r, 5.550410866482158e-2);
    s = fma(s, r, 2.4022650695910072e-1);
    s = fma(s, r, 6.9314718055994531e-1);
    s = fma(s, r, 1.0);
    return fma(s, __hiloint2double(none ? 0 : __double2hiint(pw) + ((n >> 5) << 20), __double2loint(pw)), sum);
}

// Sums of weights below this are none.
constexpr double TV_NONE = 0x1p-600;

// How far row_mass() is off, of its value, and left_mass(), of 1, at most.  With y the exponent of an entry: three F32 roundings
// of y, on average over the entries by weight below log2(V) = 22 (their entropy), 22 * 3 * 2^-24 * ln 2; 2^-22 of ex2, and of each
// of some 7 steps to a larger maximum; 16 F32 additions: less than 2^-17.  left_mass() has the row's sum in it, and its own exponentials.
constexpr float TV_CLOSE = 0x1p-16f;

// LT, DT: types of logits and drafts (DT -1: fixed choices)
template <int LT, int DT>
struct Walk {
    const TreeVerifyParams & p;
    TvShared &               sh;
    double *                 sums;  // of the CTA's chunks
    const char *             lrow;  // the current node's rows
    const char *             qrow;
    int                      lo, hi, n_ranks, n_warps;  // the CTA's slice
    int                      rank, turn, tid, lane, warp;
    bool                     held;  // a chunk a warp at most: kept from pass to pass
    double                   power;
    float                    x[TV_E], q[DT >= 0 ? TV_E : 1];

    // the chunk from i0 on
    __device__ __forceinline__ void load(float (&v)[TV_E], int i0) const {
        if (i0 + TV_CHUNK <= hi) {
            const char * at = lrow + (int64_t) (i0 + lane) * (LT == KV_F32 ? 4 : 2);
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                v[e] = load1<LT>(at, e * 32);
            }
        } else {
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                const int i = i0 + e * 32 + lane;
                v[e]        = i < hi ? load1<LT>(lrow, i) : -INFINITY;
            }
        }
    }

    static __device__ __forceinline__ void clean(float (&v)[TV_E]) {
#pragma unroll
        for (int e = 0; e < TV_E; e++) {
            v[e] = clean_logit(v[e]);
        }
    }

    __device__ __forceinline__ void load_drafts(int i0) {
        if constexpr (DT >= 0) {
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                const int i = i0 + e * 32 + lane;
                q[e]        = i < hi ? load1<DT>(qrow, i) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                q[e] = clean_draft(q[e]);
            }
        }
    }

    __device__ __forceinline__ void load_both(int i0) {
        load(x, i0);
        load_drafts(i0);
        clean(x);
    }

    // brings the slice's part of a row to L2: the passes then wait for L2 only, a few thousand bytes at a time
    __device__ __forceinline__ void fetch(const char * row, int esz) const {
        const uint64_t from = (reinterpret_cast<uint64_t>(row) + (uint64_t) lo * esz + 15) & ~15ull, to = (reinterpret_cast<uint64_t>(row) + (uint64_t) hi * esz) & ~15ull;
        if (tid == 0 && from < to) {
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"((uint32_t) (to - from)) : "memory");
        }
    }

    // the sum of a value of every thread over the cluster, the same in every thread
    __device__ __forceinline__ double total(double a) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
        }
        __syncthreads();  // (what the call before read has been read)
        if (lane == 0) {
            sh.warp_a[warp] = a;
        }
        __syncthreads();
        a = lane < n_warps ? sh.warp_a[lane] : 0.0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, d);
        }
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_a[turn] = a;
            }
            cluster_sync();
            a = lane < n_ranks ? ld_rank_f64(&sh.rank_a[turn], lane) : 0.0;
#pragma unroll
            for (int d = TV_RANKS / 2; d > 0; d >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, d);
            }
            a = __shfl_sync(0xffffffffu, a, 0);
            turn ^= 1;
        }
        return a;
    }

    // (m, sum of 2^((x - m) / t)) of each lane, joined over the warp
    __device__ __forceinline__ void join(float & m, double & z) const {
        const float a = (float) p.inv_t;
        float       top = m;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        }
        z = m > -INFINITY ? z * (double) power2((m - top) * a) : 0.0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, d);
        }
        m = top;
    }

    // (m, sum of 2^((x - m) / t)) over the row
    __device__ __forceinline__ void row_mass(float & m, double & z) {
        const float a = (float) p.inv_t;
        float       from = -INFINITY;  // what the sum is relative to: near the maximum so far, so that it seldom moves
        double      s = 0.0;
        m = -INFINITY;
        auto add = [&](const auto &... v) {  // a chunk, or two
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                ((top = fmaxf(top, v[e])), ...);
            }
            if ((top - from) * a > 8.0f) {  // (at first too)
                s *= (double) power2((from - top) * a);
                from = top;
            }
            m = fmaxf(m, top);
            if (from > -INFINITY) {
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < TV_E; e++) {
                    ((part += power2((v[e] - from) * a)), ...);
                }
                s += (double) part;
            }
        };
        const int step = n_warps * TV_CHUNK;
        if constexpr (DT >= 0) {
            for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += step) {
                load(x, i0);
                if (held) {
                    load_drafts(i0);
                }
                clean(x);
                add(x);
            }
        } else {
            for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += 2 * step) {  // two chunks' loads in flight: 52 us against 56
                float y[TV_E];
                load(x, i0);
                load(y, i0 + step);  // (-inf behind the slice)
                clean(x);
                clean(y);
                add(x, y);
            }
        }
        z = m > from ? s * (double) power2((from - m) * a) : s;
        join(m, z);
        __syncthreads();
        if (lane == 0) {
            sh.warp_m[warp] = m, sh.warp_a[warp] = z;
        }
        __syncthreads();
        m = lane < n_warps ? sh.warp_m[lane] : -INFINITY, z = lane < n_warps ? sh.warp_a[lane] : 0.0;
        join(m, z);
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_m[turn] = m, sh.rank_a[turn] = z;
            }
            cluster_sync();
            m = lane < n_ranks ? ld_rank_f32(&sh.rank_m[turn], lane) : -INFINITY, z = lane < n_ranks ? ld_rank_f64(&sh.rank_a[turn], lane) : 0.0;
            join(m, z);
            turn ^= 1;
        }
    }

    // the lowest index of the row's largest logit (-1: none is above -inf)
    __device__ __forceinline__ int row_argmax() {
        float m = -INFINITY;
        int   at = 0x7fffffff;
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += n_warps * TV_CHUNK) {
            load(x, i0);
            clean(x);
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                if (x[e] > m) {
                    m = x[e], at = i0 + e * 32 + lane;
                }
            }
        }
        auto join = [&] {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                const float y = __shfl_xor_sync(0xffffffffu, m, d);
                const int   i = __shfl_xor_sync(0xffffffffu, at, d);
                if (y > m || (y == m && i < at)) {
                    m = y, at = i;
                }
            }
        };
        join();
        __syncthreads();
        if (lane == 0) {
            sh.warp_m[warp] = m, sh.warp_i[warp] = at;
        }
        __syncthreads();
        m = lane < n_warps ? sh.warp_m[lane] : -INFINITY, at = lane < n_warps ? sh.warp_i[lane] : 0x7fffffff;
        join();
        if (n_ranks > 1) {
            if (tid == 0) {
                sh.rank_m[turn] = m, sh.rank_i[turn] = at;
            }
            cluster_sync();
            m = lane < n_ranks ? ld_rank_f32(&sh.rank_m[turn], lane) : -INFINITY, at = lane < n_ranks ? ld_rank_i32(&sh.rank_i[turn], lane) : 0x7fffffff;
            join();
            turn ^= 1;
        }
        return m > -INFINITY ? at : -1;
    }

    // sum of max(p - c q, 0), in F32 terms
    __device__ __forceinline__ double left_mass(float m, float iz, float c) {
        const float a = (float) p.inv_t;
        double      sum = 0.0;
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += n_warps * TV_CHUNK) {
            if (!held) {
                load_both(i0);
            }
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                s += fmaxf(power2((x[e] - m) * a) * iz - c * q[DT >= 0 ? e : 0], 0.0f);
            }
            sum += (double) s;
        }
        return total(sum);
    }

    // sum + 2^((v - m) / t), sum where that is below 2^-800 (or so near 0 that no sum changes by it).  By whole warps.
    __device__ __forceinline__ double add_weight(float v, float m, double sum) const {
        const bool in = (v - m) * (float) p.inv_t > -800.0f;
        return add_power((double) (in ? v : m) - (double) m, p.inv_t, power, !in, sum);
    }

    // 2^((v - m) / t), 0 where that is below 2^-800 (a token of -inf is never accepted, with a number of 0 either).  By whole warps.
    __device__ __forceinline__ double weight(float v, float m) const {
        return (v - m) * (float) p.inv_t > -800.0f ? add_weight(v, m, 0.0) : 0.0;
    }

    // what is left of the chunk's entry e: max(p - c q, 0), or the weight of a token that was not rejected.  By whole warps.
    __device__ __forceinline__ double left(int e, float m, double iz, double c) const {
        const double w = add_weight(x[e], m, 0.0);
        return DT >= 0 && c > 0.0 ? fmax(w * iz - c * (double) q[DT >= 0 ? e : 0], 0.0) : w;
    }

    // the chunk from i0 on for `left`: the rejected tokens of fixed choices count as -inf
    __device__ __forceinline__ void load_left(int i0, int n_gone) {
        if (!held || DT < 0) {
            load_both(i0);
        }
        for (int k = 0; DT < 0 && k < n_gone; k++) {
            const int at = sh.gone[k] - i0;
            if (at >= 0 && at < TV_CHUNK && (at & 31) == lane) {
#pragma unroll
                for (int e = 0; e < TV_E; e++) {
                    x[e] = e == at >> 5 ? -INFINITY : x[e];
                }
            }
        }
    }

    // sum of `left` over the row; the sums of the CTA's chunks are kept
    __device__ __forceinline__ double left_sums(float m, double iz, double c, int n_gone) {
        double sum = 0.0;
        __syncthreads();
        for (int i0 = lo + warp * TV_CHUNK; i0 < hi; i0 += n_warps * TV_CHUNK) {
            load_left(i0, n_gone);
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < TV_E; e++) {
                s = DT < 0 ? add_weight(x[e], m, s) : s + left(e, m, iz, c);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, d);
            }
            if (lane == 0) {
                sums[(i0 - lo) / TV_CHUNK] = s;
            }
            sum += lane == 0 ? s : 0.0;
        }
        return total(sum);
    }

    __device__ __forceinline__ double prefix(double s) const {  // over the lanes up to this one
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, s, d);
            s += lane >= d ? y : 0.0;
        }
        return s;
    }

    // the first entry at which the sum of what is left exceeds u times all of it, by the CTA that holds it; the chunks'
    // sums of the last left_sums() are in place
    __device__ __forceinline__ void sample(float u, float m, double iz, double c, int n_gone, int * out) {
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
        if (n_ranks > 1) {
            cluster_sync();
        } else {
            __syncthreads();
        }
        if (warp != 0) {
            return;
        }
        const double r = lane < n_ranks ? ld_rank_f64(&sh.rank_a[turn], lane) : 0.0, upto = prefix(r), all = __shfl_sync(0xffffffffu, upto, 31);
        const double target = (double) fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f) * all;
        const unsigned has = __ballot_sync(0xffffffffu, r > TV_NONE), past = __ballot_sync(0xffffffffu, r > TV_NONE && upto > target);
        // (a rounding could leave the target at the very end: the last that holds anything)
        const int owner = past ? __ffs(past) - 1 : 31 - __clz(has);
        if (has == 0 || owner != rank) {
            return;
        }
        double start = past ? __shfl_sync(0xffffffffu, upto - r, owner) : -INFINITY;
        int    chunk = -1, last = 0;
        for (int k0 = 0; k0 < n_chunks && chunk < 0; k0 += 32) {
            const double   v = k0 + lane < n_chunks ? sums[k0 + lane] : 0.0, s = prefix(v);
            const unsigned over = __ballot_sync(0xffffffffu, v > TV_NONE && start + s > target), some = __ballot_sync(0xffffffffu, v > TV_NONE);
            last = some ? k0 + 31 - __clz(some) : last;
            if (over) {
                chunk = k0 + __ffs(over) - 1;
                start += __shfl_sync(0xffffffffu, s - v, __ffs(over) - 1);
            } else {
                start += __shfl_sync(0xffffffffu, s, 31);
            }
        }
        if (chunk < 0) {
            chunk = last, start = -INFINITY;
        }
        const int i0 = lo + chunk * TV_CHUNK;
        held         = false;  // (the chunk need not be this warp's)
        load_left(i0, n_gone);
        int token = -1, backup = 0;
#pragma unroll
        for (int e = 0; e < TV_E; e++) {
            const double   v = left(e, m, iz, c), s = prefix(v);
            const unsigned over = __ballot_sync(0xffffffffu, v > TV_NONE && start + s > target), some = __ballot_sync(0xffffffffu, v > TV_NONE);
            token  = token < 0 && over ? i0 + e * 32 + __ffs(over) - 1 : token;
            backup = some ? i0 + e * 32 + 31 - __clz(some) : backup;
            start += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) {
            *out = token >= 0 ? token : backup;
        }
    }
};

template <int LT, int DT>
__global__ void __launch_bounds__(TV_THREADS, 1) tree_verify_kernel(const TreeVerifyParams p, int n_ranks, int ahead) {
    kv8_dep_wait();
    extern __shared__ double tv_sums[];
    __shared__ TvShared      sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = p.t.max_nodes;
    const int tree = (int) blockIdx.x / n_ranks;
    const int rank = n_ranks > 1 ? (int) cluster_rank() : 0;
    const int n    = tree_nodes(p.t, tree);
    int * path     = p.path + (int64_t) tree * T;
    if (n == 0) {
        if (rank == 0) {
            for (int i = tid; i < T; i += (int) blockDim.x) {
                path[i] = -1;
            }
            if (tid == 0) {
                p.n_path[tree] = 0, p.token[tree] = -1;
            }
        }
        return;
    }
    const char * lbase = p.logits.data + (int64_t) tree * p.logits.nb2, *qbase = DT >= 0 ? p.draft.data + (int64_t) tree * p.draft.nb2 : nullptr;
    for (int i = tid; i < n; i += (int) blockDim.x) {
        const int pr = tree_parent(p.t, tree, i), x = p.tokens[(int64_t) tree * T + i];
        const bool ok = i > 0 && pr >= 0 && x >= 0 && x < p.V;  // a token outside the vocabulary is never accepted
        sh.par[i] = ok ? pr : -1, sh.tok[i] = x, sh.u[i] = p.accept[(int64_t) tree * T + i];
        sh.lx[i] = ok ? clean_logit(load1<LT>(lbase + (int64_t) pr * p.logits.nb1, x)) : -INFINITY;
        sh.qx[i] = 1.0f;
        if (DT >= 0) {
            sh.qx[i] = ok ? clean_draft(load1<DT>(qbase + (int64_t) pr * p.draft.nb1, x)) : 0.0f;
        }
    }
    if (tid == 0) {
        sh.path[0] = 0;
    }  // (a row's pass has barriers before any of these are read)
    // slices of whole chunks
    const int chunks = (p.V + TV_CHUNK - 1) / TV_CHUNK, each = (chunks + n_ranks - 1) / n_ranks, n_warps = (int) blockDim.x / 32;
    Walk<LT, DT> w{ p, sh, tv_sums, lbase, qbase, min(rank * each * TV_CHUNK, p.V), min((rank + 1) * each * TV_CHUNK, p.V), n_ranks, n_warps, rank, 0, tid, lane, warp,
                    each <= n_warps, exp2((double) lane / 32.0) };
    int    cur = 0, n_path = 1, n_gone, n_no, best = -1;
    float  m = 0.0f;
    double z = 0.0;
    const bool greedy = p.inv_t == 0.0;
    constexpr int ESZ = LT == KV_F32 ? 4 : 2;
    // The walk from node `cur` on, by F32 exponentials; false: it has come to a decision that is too near to its border for them.
    // `exact`: by F64 ones.  (One after the other, and not the second's passes within the first, for the registers of its loop over
    // a row: 64 trees of 150001 tokens took 60 us that way, and 68 with the passes in a function, for 55.)
    auto walk = [&](auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
        for (;;) {
            w.lrow = lbase + (int64_t) cur * p.logits.nb1;
            w.qrow = DT >= 0 ? qbase + (int64_t) cur * p.draft.nb1 : nullptr;
            n_gone = n_no = 0;
            if (!w.held) {
                w.fetch(w.lrow, ESZ);
            }
            if (greedy) {
                best = w.row_argmax();
            } else {
                w.row_mass(m, z);
                best = m > -INFINITY ? 0 : -1;
            }
            int         next = -1;
            float       c = 0.0f, M = 1.0f, c_off = 0.0f, M_off = 0.0f;  // and how far these may be off
            const float izf = (float) (1.0 / z);
            double      iz = 1.0, cx = 0.0, Mx = 1.0;  // EXACT: 1 / the row's sum, c, M (fixed choices: what is left of the row's sum)
            if (EXACT && best >= 0) {
                const double sum = w.left_sums(m, 1.0, 0.0, 0);
                iz = 1.0 / sum, Mx = DT >= 0 ? 1.0 : sum;
            }
            bool first = true;
            for (int k0 = cur / 32 * 32; best >= 0 && next < 0 && k0 < n; k0 += 32) {
                unsigned kids = __ballot_sync(0xffffffffu, k0 + lane < n && k0 + lane > cur && sh.par[min(k0 + lane, TREE_MAX - 1)] == cur);
                while (kids && next < 0) {
                    const int i = k0 + __ffs(kids) - 1;
                    kids &= kids - 1;
                    if (greedy) {
                        next = sh.tok[i] == best ? i : -1;
                        continue;
                    }
                    if (ahead && first) {
                        // (few trees: the likeliest next row comes nearer while this one is decided on)
                        w.fetch(lbase + (int64_t) i * p.logits.nb1, ESZ);
                        first = false;
                    }
                    bool gone = false;
                    for (int k = 0; DT < 0 && k < n_gone; k++) {
                        gone = gone || sh.gone[k] == sh.tok[i];
                    }
                    const float q = sh.qx[i], u = sh.u[i];
                    float       px = 0.0f;
                    bool        taken;
                    if constexpr (EXACT) {
                        const double wx = gone ? 0.0 : w.weight(sh.lx[i], m), uq = (double) u * (double) q;
                        taken = uq * Mx < (DT >= 0 ? fmax(wx * iz - cx * (double) q, 0.0) : wx);
                    } else {
                        px = gone ? 0.0f : power2((sh.lx[i] - m) * (float) p.inv_t) * izf;
                        const float d = fmaxf(px - c * q, 0.0f) - u * q * M;
                        // (px: 2^-17 of the row's sum, 126 * 3 * 2^-24 * ln 2 of its exponent, 2^-22 of ex2, and all of it below
                        // 2^-126; 2^-22: the roundings of d)
                        if (!gone && !(fabsf(d) > 0x1p-15f * px + c_off * q + M_off * fabsf(u * q) + 0x1p-22f * (c * q + fabsf(u * q) * M) + 0x1p-125f)) {
                            return false;
                        }
                        taken = d > 0.0f;
                    }
                    if (taken) {
                        next = i;
                        continue;
                    }
                    n_no++;
                    if (DT < 0 && !gone) {
                        __syncthreads();
                        if (tid == 0) {
                            sh.gone[n_gone] = sh.tok[i];
                        }
                        __syncthreads();
                        n_gone++;
                    }
                    if constexpr (EXACT) {
                        if (DT >= 0 || !gone) {
                            cx += DT >= 0 ? Mx : 0.0;
                            Mx = w.left_sums(m, iz, cx, n_gone);
                        }
                    } else if constexpr (DT >= 0) {
                        c += M, c_off += M_off + 0x1p-23f * c;
                        M = (float) w.left_mass(m, izf, c), M_off = TV_CLOSE + c_off;  // (sum of q where p > c q: 1 / c at most, and c is 1 at least)
                    } else {
                        M = fmaxf(M - px, 0.0f), M_off += TV_CLOSE * px + 0x1p-23f;
                    }
                }
            }
            if (next < 0) {
                return true;
            }
            cur = next;
            if (tid == 0) {
                sh.path[n_path] = cur;
            }
            n_path++;
        }
    };
    if (!walk(std::false_type())) {
        walk(std::true_type());
    }
    if (!greedy && best >= 0) {
        // in F64, with drafts, the row's sum and the M again, then what is left; the target's own distribution, where nothing is
        const int last = DT >= 0 ? n_no : 0;
        double    iz = 1.0, c = 0.0;
        for (int k = 0;; k++) {
            const double sum = w.left_sums(m, iz, c, n_gone);
            if (k < last) {
                iz = k == 0 ? 1.0 / sum : iz;
                c += k == 0 ? 1.0 : sum;
            } else if (sum > TV_NONE || (c == 0.0 && n_gone == 0)) {
                break;
            } else {
                c = 0.0, n_gone = 0;
            }
        }
        w.sample(p.sample[tree], m, iz, c, n_gone, p.token + tree);
    } else if (rank == 0 && tid == 0) {
        p.token[tree] = best;
    }
    __syncthreads();
    if (rank == 0) {
        for (int i = tid; i < T; i += (int) blockDim.x) {
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
cudaError_t launch_one(const TreeVerifyParams & p, int sms, cudaStream_t stream) {
    static Kv8Once once;
    cudaError_t    e = once.smem(tree_verify_kernel<LT, DT>, 160 << 10);
    if (e != cudaSuccess) {
        return e;
    }
    // CTAs of a tree: up to 8 (the portable size), 8 chunks each or more.  Their threads: a warp for each chunk, up to what
    // lets all trees run at once at 1024 threads an SM (64 registers each), but 8 warps at least
    const int chunks  = (p.V + TV_CHUNK - 1) / TV_CHUNK;
    int       n_ranks = 1;
    while (n_ranks < TV_RANKS && chunks >= 16 * n_ranks) {
        n_ranks *= 2;
    }
    const int     each = (chunks + n_ranks - 1) / n_ranks;
    const int64_t room = (int64_t) TV_WARPS * (sms * 7 / 8) / ((int64_t) p.t.n_tree * n_ranks);  // (clusters do not fill the last SMs of a GPC)
    int           n_warps = 8;
    while (n_warps < TV_WARPS && n_warps < each && 2 * n_warps <= room) {
        n_warps *= 2;
    }
    const bool          ahead = (int64_t) p.t.n_tree * n_ranks <= sms;
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim          = dim3((unsigned) (p.t.n_tree * n_ranks));
    cfg.blockDim         = dim3((unsigned) (32 * n_warps));
    cfg.dynamicSmemBytes = (size_t) each * sizeof(double);
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
    return cudaLaunchKernelEx(&cfg, tree_verify_kernel<LT, DT>, p, n_ranks, ahead ? 1 : 0);
}

template <int LT>
cudaError_t launch_l(const TreeVerifyParams & p, int sms, cudaStream_t stream) {
    if (!p.draft.data) {
        return launch_one<LT, -1>(p, sms, stream);
    }
    switch (p.draft.type) {
        case KV_F32:
            return launch_one<LT, KV_F32>(p, sms, stream);
        case KV_F16:
            return launch_one<LT, KV_F16>(p, sms, stream);
        default:
            return launch_one<LT, KV_BF16>(p, sms, stream);
    }
}

}  // namespace

cudaError_t launch_tree_verify(const TreeVerifyParams & p, int sms, cudaStream_t stream) {
    switch (p.logits.type) {
        case KV_F32:
            return launch_l<KV_F32>(p, sms, stream);
        case KV_F16:
            return launch_l<KV_F16>(p, sms, stream);
        default:
            return launch_l<KV_BF16>(p, sms, stream);
    }
}

}  // namespace mm3fa
