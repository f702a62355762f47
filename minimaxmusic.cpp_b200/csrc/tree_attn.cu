// tree_attn.cu - attention of a tree of drafted tokens over a slab cache, on CUDA cores (sm_100a).
//
//   out[i, h] = softmax_j(scale * q[i, h] . k[j]) v[j],   j < L, and L + j' for j' = i and its ancestors
//
// One CTA of 4 warps takes up to 4 query heads of a kv head for one node, so that a K and a V row is read once for
// them.  Eight lanes share a key (D / 8 elements each): a dot is 3 shuffles, and each of the 16 groups of eight lanes
// keeps a running maximum, sum and output of its keys; the groups are joined at the end, in their order.  Keys that the
// node does not see are not read.  Every type is widened to F32 exactly, all arithmetic is F32.
//
// Bound: issue and the latency of its loads, a node's keys one after another: two sequences of 8192, 24 nodes, 32 heads on 8,
// D = 128, F32 slabs take 2438 us, 300 tokens and 5 nodes 39.  For slabs and head sizes that the tensor cores do not take
// (there 32 us at 8192 from F16, 17 at 300).  Its work is not split over a unit's keys, so that one node takes 1548 us at 8192, where
// the decode kernels, with the tree as a mask, take 57; Q8_0 832 and 74, 4 nodes 841 and 32.
#include "tree.cuh"

namespace mm3fa {

namespace {

constexpr int TA_THREADS = 128;
constexpr int TA_GROUPS  = TA_THREADS / 8;

// elements [e0, e0 + 8) of a row, e0 a multiple of 8
__device__ __forceinline__ void load8(const char * row, int type, int e0, bool vec, float (&x)[8]) {
    if (type == KV_Q8_0) {
        const char *     b = row + (e0 / QK8_0) * Q8_0_BLOCK;
        const float      d = __half2float(*reinterpret_cast<const __half *>(b));
        const uint16_t * c = reinterpret_cast<const uint16_t *>(b + 2 + e0 % QK8_0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint16_t w = c[i];
            x[2 * i]         = d * (float) (int8_t) (w & 0xff);
            x[2 * i + 1]     = d * (float) (int8_t) (w >> 8);
        }
        return;
    }
    uint32_t  w[8];
    const int n = type == KV_F32 ? 8 : 4;
    const char * at = row + (int64_t) e0 * (type == KV_F32 ? 4 : 2);
    if (vec) {
        const uint4 a = *reinterpret_cast<const uint4 *>(at);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        if (n == 8) {
            const uint4 b = *reinterpret_cast<const uint4 *>(at + 16);
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        }
    } else if (n == 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            w[i] = reinterpret_cast<const uint32_t *>(at)[i];
        }
    } else {
        const uint16_t * h = reinterpret_cast<const uint16_t *>(at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = h[2 * i] | (uint32_t) h[2 * i + 1] << 16;
        }
    }
    if (n == 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = __uint_as_float(w[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = type == KV_F16 ? h2_to_f2(w[i]) : bf2_to_f2(w[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

// D = 64 C; R: query heads of a CTA
template <int C, int R>
__global__ void __launch_bounds__(TA_THREADS) tree_attn_kernel(const TreeAttnParams p) {
    kv8_dep_wait();
    constexpr int      D = 64 * C;
    __shared__ uint8_t on_path[TREE_MAX];
    __shared__ float   gm[TA_GROUPS][R], gl[TA_GROUPS][R];
    __shared__ float   go[TA_GROUPS][D];
    const int tid = threadIdx.x, lane8 = tid & 7, group = tid >> 3;
    const int per = (p.ratio + R - 1) / R, hk = (int) blockIdx.y / per, g0 = (int) blockIdx.y % per * R;
    const int i = blockIdx.x, s = blockIdx.z, tree = s % p.t.n_tree, n = tree_nodes(p.t, tree);
    if (i >= n) {
        return;
    }
    const int L = min(max(p.kv_len[s], 0), p.n_kv);
    for (int j = tid; j < TREE_MAX; j += TA_THREADS) {
        on_path[j] = 0;
    }
    __syncthreads();
    if (tid == 0) {
        for (int a = i; a >= 0; a = tree_parent(p.t, tree, a)) {
            on_path[a] = 1;
        }
    }
    __syncthreads();
    float q[R][8 * C], acc[R][8 * C], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int    h   = hk * p.ratio + min(g0 + r, p.ratio - 1);
        const char * row = p.q.data + (int64_t) i * p.q.nb1 + (int64_t) h * p.q.nb2 + (int64_t) s * p.q.nb3;
        m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            float x[8];
            load8(row, p.q.type, (c * 8 + lane8) * 8, p.q.vec, x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                q[r][c * 8 + e] = x[e], acc[r][c * 8 + e] = 0.0f;
            }
        }
    }
    const char * kb = p.k.data + (int64_t) hk * p.k.nb2 + (int64_t) s * p.k.nb3;
    const char * vb = p.v.data + (int64_t) hk * p.v.nb2 + (int64_t) s * p.v.nb3;
    const int    n_keys = min(L + i + 1, p.n_kv);  // a node's ancestors come before it
    // whole warps go round together: the shuffles below want all lanes
    for (int j0 = 0; j0 < n_keys; j0 += TA_GROUPS) {
        const int  j    = j0 + group;
        const bool seen = j < n_keys && (j < L || on_path[j - L]);
        float      sc[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            sc[r] = 0.0f;
        }
        if (seen) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                float x[8];
                load8(kb + (int64_t) j * p.k.nb1, p.k.type, (c * 8 + lane8) * 8, p.k.vec, x);
#pragma unroll
                for (int r = 0; r < R; r++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        sc[r] = fmaf(q[r][c * 8 + e], x[e], sc[r]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int d = 1; d < 8; d *= 2) {
                sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], d);
            }
        }
        if (!seen) {
            continue;
        }
        float w[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            float x = sc[r] * p.scale;
            if (p.softcap > 0.0f) {
                x = p.softcap * tanhf(x / p.softcap);
            }
            const float top = fmaxf(m[r], x), grow = m[r] == top ? 1.0f : expf(m[r] - top);
            w[r] = x == -INFINITY ? 0.0f : expf(x - top);
            l[r] = l[r] * grow + w[r], m[r] = top;
#pragma unroll
            for (int e = 0; e < 8 * C; e++) {
                acc[r][e] *= grow;
            }
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            float x[8];
            load8(vb + (int64_t) j * p.v.nb1, p.v.type, (c * 8 + lane8) * 8, p.v.vec, x);
#pragma unroll
            for (int r = 0; r < R; r++) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    acc[r][c * 8 + e] = fmaf(w[r], x[e], acc[r][c * 8 + e]);
                }
            }
        }
    }
    // join the groups, one query head after another
    if (lane8 == 0) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            gm[group][r] = m[r], gl[group][r] = l[r];
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; c++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                go[group][(c * 8 + lane8) * 8 + e] = acc[r][c * 8 + e];
            }
        }
        __syncthreads();
        if (g0 + r >= p.ratio) {
            continue;
        }
        float top = -INFINITY, sum = 0.0f, f[TA_GROUPS];
#pragma unroll
        for (int g = 0; g < TA_GROUPS; g++) {
            top = fmaxf(top, gm[g][r]);
        }
#pragma unroll
        for (int g = 0; g < TA_GROUPS; g++) {  // (a sum of NaN passes through)
            f[g] = gl[g][r] == 0.0f ? 0.0f : (gm[g][r] == top ? 1.0f : expf(gm[g][r] - top));
            sum += gl[g][r] * f[g];
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int   h   = hk * p.ratio + g0 + r;
        char *      out = p.o.data + (int64_t) h * p.o.nb1 + (int64_t) i * p.o.nb2 + (int64_t) s * p.o.nb3;
        for (int e = tid; e < D; e += TA_THREADS) {
            float o = 0.0f;
#pragma unroll
            for (int g = 0; g < TA_GROUPS; g++) {
                o = gl[g][r] == 0.0f ? o : fmaf(go[g][e], f[g], o);
            }
            o *= inv;
            if (p.o.type == KV_F32) {
                reinterpret_cast<float *>(out)[e] = o;
            } else if (p.o.type == KV_F16) {
                reinterpret_cast<__half *>(out)[e] = __float2half_rn(o);
            } else {
                reinterpret_cast<__nv_bfloat16 *>(out)[e] = __float2bfloat16_rn(o);
            }
        }
    }
}

template <int C, int R>
cudaError_t launch_one(const TreeAttnParams & p, cudaStream_t stream) {
    const dim3 grid((unsigned) p.t.max_nodes, (unsigned) (p.n_head_kv * ((p.ratio + R - 1) / R)), (unsigned) p.n_seq);
    return kv8_launch(tree_attn_kernel<C, R>, grid, TA_THREADS, 0, stream, p);
}

}  // namespace

cudaError_t launch_tree_attn(const TreeAttnParams & p, cudaStream_t stream) {
    switch (p.D) {
        case 64:
            return launch_one<1, 4>(p, stream);
        case 128:
            return launch_one<2, 4>(p, stream);
        default:
            return launch_one<4, 2>(p, stream);
    }
}

}  // namespace mm3fa
