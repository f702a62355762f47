// kv8_pages.cu - fork, compact and reserve the pages of the 8-bit paged KV cache (sm_100a).
//
// A plan kernel of one CTA counts, ranks and assigns pages with block-wide scans (no order depends on
// timing: fresh pages are the free ones with the lowest numbers, given out in order of sequence and
// page slot), and writes the reference counts, the changed table rows and the list of page copies.
// A copy kernel over the whole GPU then moves the listed pages of every layer and the rest of the
// table.  Sources are pages that were live before the call, destinations pages that were free, so no
// copy reads what another writes.
//
// The plan is latency: one CTA, since every rank needs the counts before it (9 to 10 us with the copy, for 16
// sequences of up to 700 tokens).  The copy is memory: deep copies of 3 of 8 sequences of 900 to 2500 tokens in 36 layers
// (0.77 GB read and written) take 155 us, 76 % of the copy bandwidth of 6.54 TB/s, in a graph over three caches in turn, and 124 to
// 141 as calls on one; moving half of a pool of such 88, 79 %.
//
// A call that finds too few free pages changes nothing and leaves a bit in the workspace's status.
#include "kv8.cuh"

#include <climits>

namespace mm3fa {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_ITEMS   = 8;  // page counts per thread and scan step
constexpr int COPY_THREADS = 256;
constexpr int COPY_UNROLL  = 8;  // 16-byte words in flight per thread

// Exclusive block scan of one int per thread; `total` gets the sum.  red: 33 shared ints.
__device__ __forceinline__ int plan_scan(int x, int & total, int * red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int       v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        v += lane >= o ? u : 0;
    }
    __syncthreads();  // red may still be read from the scan before
    if (lane == 31) {
        red[warp] = v;
    }
    __syncthreads();
    if (warp == 0) {
        int w = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            w += lane >= o ? u : 0;
        }
        red[lane] = w;
    }
    __syncthreads();
    total = red[31];
    return v - x + (warp ? red[warp - 1] : 0);
}

// Exclusive scan of need[0 .. n) into off; returns the total.
__device__ int plan_offsets(const int * need, int * off, int n, int * red) {
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const int i = i0 + (int) threadIdx.x;
        int       total;
        const int at = plan_scan(i < n ? need[i] : 0, total, red);
        if (i < n) {
            off[i] = base + at;
        }
        base += total;
    }
    return base;
}

// Writes the first `want` free pages (refs 0) in ascending order to list; returns how many there are
// (counting may stop once there are enough).
__device__ int plan_free_pages(const int * refs, int n_pages, int want, int * list, int * red) {
    int found = 0;
    for (int b = 0; b < n_pages && found < want; b += PLAN_THREADS * PLAN_ITEMS) {
        const int i0   = b + (int) threadIdx.x * PLAN_ITEMS;
        int       free = 0;
#pragma unroll
        for (int k = 0; k < PLAN_ITEMS; k++) {
            free |= (i0 + k < n_pages && refs[i0 + k] == 0) ? 1 << k : 0;
        }
        int total;
        int at = found + plan_scan(__popc(free), total, red);
#pragma unroll
        for (int k = 0; k < PLAN_ITEMS; k++) {
            if (free >> k & 1) {
                if (at < want) {
                    list[at] = i0 + k;
                }
                at++;
            }
        }
        found += total;
    }
    return found;
}

__device__ __forceinline__ bool plan_valid(int page, int n_pages) {
    return (unsigned) page < (unsigned) n_pages;
}

__global__ void __launch_bounds__(PLAN_THREADS) kv8_fork_plan_kernel(const Kv8PlanParams p) {
    __shared__ int red[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = PLAN_THREADS / 32;
    kv8_dep_wait();
    // win[d]: the first pair that names sequence d as its destination
    for (int d = tid; d < p.n_seq; d += PLAN_THREADS) {
        p.win[d] = INT_MAX;
    }
    for (int i = tid; i < p.n_pages; i += PLAN_THREADS) {
        p.refs_out[i] = p.refs_in[i];
    }
    __syncthreads();
    for (int i = tid; i < p.n_pairs; i += PLAN_THREADS) {
        const int d = p.dst[i], s = p.src ? p.src[i] : -1;
        if (d >= 0 && d < p.n_seq && s >= -1 && s < p.n_seq) {
            atomicMin(&p.win[d], i);
        }
    }
    __syncthreads();
    // off[d]: how many fresh pages sequence d takes.  win[d] becomes its source, -1 (emptied) or -2 (unchanged)
    for (int d = warp; d < p.n_seq; d += warps) {
        const int i = p.win[d];
        int       s = i == INT_MAX ? -2 : (p.src ? p.src[i] : -1);
        s           = s == d ? -2 : s;
        int need    = 0;
        if (s >= 0) {
            const int n  = min(max(p.len_in[s], 0), p.max_pages * p.P);
            const int np = (n + p.P - 1) / p.P;
            for (int j = (p.deep ? 0 : n / p.P) + lane; j < np; j += 32) {
                need += plan_valid(p.table_in[(int64_t) s * p.in_stride + j], p.n_pages);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                need += __shfl_xor_sync(0xffffffffu, need, o);
            }
        }
        __syncwarp();
        if (lane == 0) {
            p.win[d] = s;
            p.off[d] = need;
        }
    }
    __syncthreads();
    const int total = plan_offsets(p.off, p.off, p.n_seq, red);
    const int found = plan_free_pages(p.refs_in, p.n_pages, total, p.copy_dst, red);
    __syncthreads();
    const bool failed = found < total;
    if (tid == 0) {
        p.head[KV8_WS_COPIES] = failed ? 0 : total;
        p.head[KV8_WS_FAILED] = failed;
        if (failed) {
            kv8_report(p.status, ST_PAGES);
        }
    }
    if (failed) {
        return;
    }
    for (int d = warp; d < p.n_seq; d += warps) {
        const int s = p.win[d];
        if (s == -2) {
            continue;
        }
        const int   n     = s < 0 ? 0 : min(max(p.len_in[s], 0), p.max_pages * p.P);
        const int   np    = (n + p.P - 1) / p.P;
        const int   first = p.deep ? 0 : n / p.P;  // pages from here on are copied
        const int * old   = p.table_in + (int64_t) d * p.in_stride;
        const int * from  = p.table_in + (int64_t) (s < 0 ? d : s) * p.in_stride;
        int *       out   = p.table_out + (int64_t) d * p.out_stride;
        int         at    = p.off[d];
        for (int j0 = 0; j0 < p.max_pages; j0 += 32) {
            const int  j    = j0 + lane;
            const bool in   = j < p.max_pages;
            const int  gone = in ? old[j] : -1;
            int        page = in && j < np ? from[j] : -1;
            const bool copy = j >= first && plan_valid(page, p.n_pages);
            if (plan_valid(gone, p.n_pages)) {
                atomicSub(&p.refs_out[gone], 1);
            }
            const uint32_t who = __ballot_sync(0xffffffffu, copy);
            if (copy) {
                const int k   = at + __popc(who & ((1u << lane) - 1u));
                const int to  = p.copy_dst[k];
                p.copy_src[k] = page;
                p.refs_out[to] = 1;
                page          = to;
            } else if (plan_valid(page, p.n_pages)) {
                atomicAdd(&p.refs_out[page], 1);
            }
            if (in) {
                out[j] = page;
            }
            at += __popc(who);
        }
    }
}

__global__ void __launch_bounds__(PLAN_THREADS) kv8_compact_plan_kernel(const Kv8PlanParams p) {
    __shared__ int red[32];
    const int tid = threadIdx.x;
    kv8_dep_wait();
    int live = 0, n_live, n_move;
    for (int i = tid; i < p.n_pages; i += PLAN_THREADS) {
        live += p.refs_in[i] > 0;
    }
    plan_scan(live, n_live, red);
    // the r-th hole in [0, n_live) takes the r-th live page from n_live on
    n_move = plan_free_pages(p.refs_in, n_live, n_live, p.copy_dst, red);
    int base = 0;
    for (int b = n_live; b < p.n_pages; b += PLAN_THREADS) {
        const int i  = b + tid;
        const int mv = i < p.n_pages && p.refs_in[i] > 0;
        int       total;
        const int at = base + plan_scan(mv, total, red);
        if (mv) {
            p.copy_src[at] = i;
        }
        base += total;
    }
    __syncthreads();
    n_move = min(n_move, base);
    for (int i = tid; i < p.n_pages; i += PLAN_THREADS) {
        p.map[i]      = i;
        p.refs_out[i] = i < n_live ? p.refs_in[i] : 0;
    }
    __syncthreads();
    for (int r = tid; r < n_move; r += PLAN_THREADS) {
        const int from = p.copy_src[r], to = p.copy_dst[r];
        p.map[from]    = to;
        p.refs_out[to] = p.refs_in[from];
    }
    if (tid == 0) {
        p.head[KV8_WS_COPIES] = n_move;
        p.head[KV8_WS_FAILED] = 0;
    }
}

__global__ void __launch_bounds__(PLAN_THREADS) kv8_reserve_kernel(const Kv8PlanParams p) {
    __shared__ int red[32];
    __shared__ int over;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = PLAN_THREADS / 32;
    kv8_dep_wait();
    if (tid == 0) {
        over = 0;
    }
    __syncthreads();
    for (int d = warp; d < p.n_seq; d += warps) {
        const int n  = max(p.n_tok[d], 0);
        int       np = (int) (((int64_t) n + p.P - 1) / p.P), need = 0;
        if (np > p.max_pages) {
            over = 1;
            np   = p.max_pages;
        }
        for (int j = lane; j < np; j += 32) {
            need += p.table_out[(int64_t) d * p.out_stride + j] < 0;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            need += __shfl_xor_sync(0xffffffffu, need, o);
        }
        if (lane == 0) {
            p.off[d] = need;
        }
    }
    __syncthreads();
    const int total = plan_offsets(p.off, p.off, p.n_seq, red);
    const int found = plan_free_pages(p.refs_out, p.n_pages, total, p.copy_dst, red);
    __syncthreads();
    if (found < total || over) {
        if (tid == 0) {
            kv8_report(p.status, ST_PAGES);
        }
        return;
    }
    for (int d = warp; d < p.n_seq; d += warps) {
        const int np = (int) (((int64_t) max(p.n_tok[d], 0) + p.P - 1) / p.P);
        int       at = p.off[d];
        for (int j0 = 0; j0 < np; j0 += 32) {
            const int      j    = j0 + lane;
            int *          e    = p.table_out + (int64_t) d * p.out_stride + j;
            const bool     want = j < np && *e < 0;
            const uint32_t who  = __ballot_sync(0xffffffffu, want);
            if (want) {
                const int page   = p.copy_dst[at + __popc(who & ((1u << lane) - 1u))];
                *e               = page;
                p.refs_out[page] = 1;
            }
            at += __popc(who);
        }
    }
}

// Copies the planned pages of every layer, K and V, with their scales, and finishes the table:
// FORK: rows that no pair changes (all of them, and all counts, where the plan failed); otherwise
// (compact) every entry through the map.
template <bool FORK>
__global__ void __launch_bounds__(COPY_THREADS) kv8_copy_kernel(const Kv8PlanParams p, const Kv8PoolCopy c) {
    kv8_dep_wait();
    const int64_t gid = (int64_t) blockIdx.x * COPY_THREADS + threadIdx.x, gsz = (int64_t) gridDim.x * COPY_THREADS;
    const int     n      = p.head[KV8_WS_COPIES];
    const bool    failed = p.head[KV8_WS_FAILED] != 0;
    // pages, in pieces of COPY_THREADS * COPY_UNROLL words
    constexpr int64_t PIECE  = (int64_t) COPY_THREADS * COPY_UNROLL * 16;
    const int64_t     pieces = (c.page_bytes + PIECE - 1) / PIECE;
    const int64_t     work   = (int64_t) n * c.n_layers * 2 * pieces;
    for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
        const int64_t piece = w % pieces, u = w / pieces;
        const int     i     = (int) (u % n);
        const int64_t lk    = u / n;  // layer * 2 + (K: 0, V: 1)
        const int64_t layer = (lk >> 1) * c.n_pages;
        char *        pool  = lk & 1 ? c.v : c.k;
        const int64_t at    = piece * PIECE + threadIdx.x * 16;
        const char *  src   = pool + (layer + p.copy_src[i]) * c.page_bytes;
        char *        dst   = pool + (layer + p.copy_dst[i]) * c.page_bytes;
        uint4         x[COPY_UNROLL];
#pragma unroll
        for (int k = 0; k < COPY_UNROLL; k++) {
            const int64_t b = at + (int64_t) k * COPY_THREADS * 16;
            if (b < c.page_bytes) {
                x[k] = __ldcs(reinterpret_cast<const uint4 *>(src + b));
            }
        }
#pragma unroll
        for (int k = 0; k < COPY_UNROLL; k++) {
            const int64_t b = at + (int64_t) k * COPY_THREADS * 16;
            if (b < c.page_bytes) {
                __stcs(reinterpret_cast<uint4 *>(dst + b), x[k]);
            }
        }
    }
    const int64_t scales = (int64_t) n * c.n_layers * c.n_head_kv;
    for (int64_t w = gid; w < scales; w += gsz) {
        const int     h  = (int) (w % c.n_head_kv);
        const int     i  = (int) (w / c.n_head_kv % n);
        const int64_t lp = w / c.n_head_kv / n * c.n_pages;
        const int64_t a = (lp + p.copy_src[i]) * c.n_head_kv + h, b = (lp + p.copy_dst[i]) * c.n_head_kv + h;
        c.k_scale[b] = c.k_scale[a];
        c.v_scale[b] = c.v_scale[a];
    }
    for (int64_t w = gid; w < (int64_t) p.n_seq * p.max_pages; w += gsz) {
        const int s = (int) (w / p.max_pages), j = (int) (w % p.max_pages);
        int       e = p.table_in[s * p.in_stride + j];
        if (FORK) {
            if (!failed && p.win[s] != -2) {
                continue;
            }
        } else {
            e = plan_valid(e, p.n_pages) ? p.map[e] : -1;
        }
        p.table_out[s * p.out_stride + j] = e;
    }
    if (FORK) {
        for (int64_t s = gid; s < p.n_seq; s += gsz) {
            const int from = failed ? -2 : p.win[s];
            p.len_out[s]   = from == -1 ? 0 : p.len_in[from < 0 ? s : from];
        }
    }
}

cudaError_t launch_kv8_fork(const Kv8PlanParams & p, const Kv8PoolCopy & c, int sms, cudaStream_t stream) {
    const cudaError_t e = kv8_launch(kv8_fork_plan_kernel, dim3(1), PLAN_THREADS, 0, stream, p);
    return e != cudaSuccess ? e : kv8_launch(kv8_copy_kernel<true>, dim3(4 * (unsigned) sms), COPY_THREADS, 0, stream, p, c);
}

cudaError_t launch_kv8_compact(const Kv8PlanParams & p, const Kv8PoolCopy & c, int sms, cudaStream_t stream) {
    const cudaError_t e = kv8_launch(kv8_compact_plan_kernel, dim3(1), PLAN_THREADS, 0, stream, p);
    return e != cudaSuccess ? e : kv8_launch(kv8_copy_kernel<false>, dim3(4 * (unsigned) sms), COPY_THREADS, 0, stream, p, c);
}

cudaError_t launch_kv8_reserve(const Kv8PlanParams & p, cudaStream_t stream) {
    return kv8_launch(kv8_reserve_kernel, dim3(1), PLAN_THREADS, 0, stream, p);
}

}  // namespace mm3fa
