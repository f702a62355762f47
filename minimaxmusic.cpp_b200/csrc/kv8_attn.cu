// kv8_attn.cu - attention over the 8-bit paged KV cache (sm_100a).
//
// One warp per (query row, head, sequence), the lanes along the head dimension, keys in turn with
// the running maximum and sum of the softmax.
#include "kv8.cuh"

namespace mm3fa {

template <int D>
__global__ void __launch_bounds__(128) kv8_attn_kernel(const Kv8AttnParams p) {
    constexpr int E = D / 32;
    kv8_dep_wait();
    const int     lane = threadIdx.x & 31;
    const int64_t w    = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5);
    const int     row  = (int) (w % p.n_q);
    const int     h    = (int) (w / p.n_q % p.n_head);
    const int64_t s64  = w / p.n_q / p.n_head;
    if (s64 >= p.t.n_seq) {
        return;
    }
    const int s  = (int) s64;
    const int nq = p.q_len ? min(p.q_len[s], p.n_q) : p.n_q;
    if (row >= nq) {
        return;
    }
    int n = min(max(p.kv_len[s], 0), p.t.max_pages * p.c.P);
    n     = p.causal ? n - (nq - 1 - row) : n;
    const char * qr = p.q.data + row * p.q.nb1 + h * p.q.nb2 + s * p.q.nb3;
    float        q[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; e++) {
        const int i = lane * E + e;
        q[e]        = p.q.type == KV_F32 ? reinterpret_cast<const float *>(qr)[i]
                    : p.q.type == KV_F16 ? __half2float(reinterpret_cast<const __half *>(qr)[i])
                                         : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(qr)[i]);
        o[e]        = 0.0f;
    }
    const int hk = h / p.ratio;
    for (int j = 0; j < n; j++) {
        const int page = kv8_page(p.t, p.c.n_pages, s, j >> p.c.log2p);
        if (page < 0) {
            continue;
        }
        const int64_t  ph = (int64_t) page * p.c.n_head_kv + hk;
        const int64_t  at = (ph * p.c.P + (j & (p.c.P - 1))) * D + lane * E;
        float          x  = 0.0f;
        for (int e = 0; e < E; e++) {
            x += q[e] * (float) p.c.k[at + e];
        }
        for (int d = 16; d; d >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, d);
        }
        x *= p.scale * p.c.k_scale[ph];
        if (p.softcap > 0.0f) {
            x = p.softcap * tanhf(x / p.softcap);
        }
        const float mn = x != x ? x : fmaxf(m, x), a = mn == -INFINITY ? 1.0f : expf(m - mn), e1 = mn == -INFINITY ? 0.0f : expf(x - mn);
        l = l * a + e1;
        for (int e = 0; e < E; e++) {
            o[e] = o[e] * a + e1 * p.c.v_scale[ph] * (float) p.c.v[at + e];
        }
        m = mn;
    }
    char * dr = p.o.data + h * p.o.nb1 + row * p.o.nb2 + s * p.o.nb3;
    for (int e = 0; e < E; e++) {
        const int   i = lane * E + e;
        const float y = l != 0.0f ? o[e] / l : 0.0f;
        if (p.o.type == KV_F32) {
            reinterpret_cast<float *>(dr)[i] = y;
        } else if (p.o.type == KV_F16) {
            reinterpret_cast<__half *>(dr)[i] = __float2half_rn(y);
        } else {
            reinterpret_cast<__nv_bfloat16 *>(dr)[i] = __float2bfloat16_rn(y);
        }
    }
}

size_t kv8_attn_workspace_bytes(int, int, int, int, int, int) {
    return WS_STATUS_BYTES;
}

cudaError_t launch_kv8_attn(const Kv8AttnParams & p, int, cudaStream_t stream) {
    const int64_t warps = (int64_t) p.n_q * p.n_head * p.t.n_seq;
    const dim3    grid((unsigned) ((warps + 3) / 4));
    switch (p.c.D) {
        case 64:
            return kv8_launch(kv8_attn_kernel<64>, grid, 128, 0, stream, p);
        case 128:
            return kv8_launch(kv8_attn_kernel<128>, grid, 128, 0, stream, p);
        default:
            return kv8_launch(kv8_attn_kernel<256>, grid, 128, 0, stream, p);
    }
}

}  // namespace mm3fa
