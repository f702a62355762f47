// kv8.cuh - the 8-bit paged KV cache: launch parameters and helpers shared by its kernels (sm_100a).
//
// The cache holds int8 codes [layer][page][kv head][token in page][dim] for K and for V and one F32
// scale per (layer, page, kv head); a value is code * scale.  A sequence's tokens sit in the pages
// its table row names, P tokens each.  Entries outside [0, n_pages) name no page: the attention
// takes their keys as absent, the append and the read skip their rows.
#pragma once

#include "fa_common.cuh"

#include <cuda_runtime.h>

#include <atomic>
#include <cstdlib>

namespace mm3fa {

constexpr uint32_t ST_PAGES = 2u;  // status bit: a page operation found too few free pages

// One layer of a cache.
struct Kv8Layer {
    int8_t * k;
    int8_t * v;
    float *  k_scale;
    float *  v_scale;
    int      n_pages, n_head_kv, D;
    int      P, log2p;  // tokens per page (a power of two)
};

struct Kv8Table {
    const int * pages;   // [n_seq][stride]
    int64_t     stride;  // entries
    int         max_pages, n_seq;
};

// Strided rows [D, rows, heads, seqs] of F32, F16 or BF16 values (ggml byte strides).
struct Kv8Rows {
    char *  data;
    int64_t nb1, nb2, nb3;
    int     type;
    int     vec;  // every row starts 16-byte aligned
};

struct Kv8StoreParams {
    Kv8Layer    c;
    Kv8Table    t;
    Kv8Rows     k, v;
    const int * start;  // [n_seq]
    const int * n;      // [n_seq] or null: n_rows
    int         n_rows;
};

struct Kv8AttnParams {
    Kv8Layer    c;
    Kv8Table    t;
    Kv8Rows     q, o;    // q [D, n_q, H, N]; o [D, H, n_q, N]
    const int * kv_len;  // [N]
    const int * q_len;   // [N] or null: n_q
    int         n_q, n_head, ratio;
    uint32_t    ratio_inv;  // floor(2^32 / ratio) + 1 (0: ratio 1)
    int         causal;
    float       scale, softcap;
    // workspace
    uint32_t *  status;
    uint32_t *  counters;
    float *     part;
    int         parts;  // of a block of rows' keys, at most (many rows)
    uint64_t    timeout_ns;
};

struct Kv8PoolCopy {
    char *   k;
    char *   v;
    float *  k_scale;
    float *  v_scale;
    int      n_layers, n_pages, n_head_kv;
    int64_t  page_bytes;  // of one layer's K or V, a multiple of 16
};

constexpr size_t KV8_WS_ZEROED = 1 << 16;  // bytes of a workspace that a caller zeroes: none is smaller

// Words of a workspace that may hold the address of a second status word (0: none): a graph that zeroes its workspace at
// every replay leaves there what its calls found.
constexpr int KV8_WS_ALSO = 4;

// Workspace of the page operations (int32 words from its base; 64 words of status and counts first).
constexpr int KV8_WS_COPIES = 32;  // page copies that the plan wants done
constexpr int KV8_WS_FAILED = 33;  // nonzero: too few pages, nothing changes
constexpr int KV8_WS_HEAD   = 64;

struct Kv8PlanParams {
    const int * table_in;
    int *       table_out;
    int64_t     in_stride, out_stride;
    int         n_seq, max_pages, n_pages, P;
    const int * len_in;
    int *       len_out;
    const int * refs_in;
    int *       refs_out;
    const int * src;  // null: every dst is emptied
    const int * dst;
    int         n_pairs;
    int         deep;
    const int * n_tok;  // reserve
    // workspace
    uint32_t *  status;
    int *       head;      // KV8_WS_HEAD words
    int *       copy_src;  // [n_pages]
    int *       copy_dst;  // [n_pages]
    int *       map;       // [n_pages]
    int *       win;       // [n_seq]
    int *       off;       // [n_seq]
};

// ------------------------------------------------------------------ device helpers

__device__ __forceinline__ void kv8_dep_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// r / d for r < 2^24 and inv = floor(2^32 / d) + 1: the error r (inv d - 2^32) / 2^32 d stays below 1 / d
// while r d < 2^32
__device__ __forceinline__ uint32_t kv8_div(uint32_t r, uint32_t inv) {
    return inv ? __umulhi(r, inv) : r;
}

// The page of a sequence's page slot j, or -1.
__device__ __forceinline__ int kv8_page(const Kv8Table & t, int n_pages, int s, int j) {
    if (j < 0 || j >= t.max_pages) {
        return -1;
    }
    const int p = t.pages[(int64_t) s * t.stride + j];
    return (unsigned) p < (unsigned) n_pages ? p : -1;
}

// Sets a bit of the workspace's status, and of the second status word where there is one.
__device__ __forceinline__ void kv8_report(uint32_t * status, uint32_t bit) {
    atomicOr(status, bit);
    const uint64_t also = status[KV8_WS_ALSO] | (uint64_t) status[KV8_WS_ALSO + 1] << 32;  // (the workspace may be 4-byte aligned)
    if (also) {
        atomicOr(reinterpret_cast<uint32_t *>(also), bit);
    }
}

// ------------------------------------------------------------------ host helpers

inline bool kv8_pdl() {
    static const bool pdl = [] {
        const char * e = std::getenv("MM3FA_PDL");
        return !(e && std::atoi(e) == 0);
    }();
    return pdl;
}

// Launches with programmatic stream serialisation (MM3FA_PDL=0 turns it off): the CTAs may start
// once the previous kernel's have exited or have let their dependents go (the peer wait does so at its entry);
// every kernel here waits with griddepcontrol.wait, for that kernel's end, before it reads anything or takes a time.
template <typename... KArgs, typename... Args>
cudaError_t kv8_launch(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim          = grid;
    cfg.blockDim         = dim3((unsigned) threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream           = stream;
    cfg.attrs            = attr;
    cfg.numAttrs         = 0;
    if (kv8_pdl()) {
        attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs                                       = 1;
    }
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// A kernel's dynamic shared memory limit, raised once per device.
struct Kv8Once {
    std::atomic<uint64_t> done{ 0 };
    template <typename Kern>
    cudaError_t smem(Kern kern, size_t bytes) {
        int         dev = 0;
        cudaError_t e   = cudaGetDevice(&dev);
        if (e != cudaSuccess) {
            return e;
        }
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (bit && (done.load(std::memory_order_acquire) & bit)) {
            return cudaSuccess;
        }
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) bytes);
        if (e == cudaSuccess) {
            done.fetch_or(bit, std::memory_order_release);
        }
        return e;
    }
};

cudaError_t launch_kv8_append(const Kv8StoreParams & p, cudaStream_t stream);
cudaError_t launch_kv8_read(const Kv8StoreParams & p, cudaStream_t stream);
cudaError_t launch_kv8_attn(const Kv8AttnParams & p, int sms, cudaStream_t stream);
cudaError_t launch_kv8_dense(const Kv8AttnParams & p, cudaStream_t stream);
int         kv8_dense_tile(const Kv8AttnParams & p);  // rows of a CTA
int         kv8_dense_parts(int64_t items, int64_t tokens, int sms);  // parts of a block of rows' keys, at most
size_t      kv8_dense_part_bytes(int D, int64_t items, int tile, int parts);
size_t      kv8_attn_workspace_bytes(int D, int64_t rows, int64_t heads, int64_t tokens, int sms);
cudaError_t launch_kv8_fork(const Kv8PlanParams & p, const Kv8PoolCopy & c, int sms, cudaStream_t stream);
cudaError_t launch_kv8_compact(const Kv8PlanParams & p, const Kv8PoolCopy & c, int sms, cudaStream_t stream);
cudaError_t launch_kv8_reserve(const Kv8PlanParams & p, cudaStream_t stream);

// defined in mm3fa_abi.cu
int      host_record_cuda(cudaError_t e);
int      host_sm_count();      // of the current device, 0 without one
int      host_device_major();  // compute capability
uint64_t host_wait_timeout_ns();

}  // namespace mm3fa
