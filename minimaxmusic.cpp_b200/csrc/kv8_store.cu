// kv8_store.cu - append to and read from the 8-bit paged KV cache (sm_100a).
//
// Append: one CTA per (page that gets new rows, kv head, K or V).  With x the new rows of the page
// and held the rows of earlier tokens in it,
//     d' = max(d if held, max|x| / 127)             (F32, the division rounded to nearest)
//     held codes  c' = rne(c * d / d')              (only where d' > d)
//     new codes   c  = clamp(rne(x / d'), -127, 127)
// with the quotients rounded as exact arithmetic would (rne: ties to even).  Values that are not
// finite do not enter the maximum; NaN is stored as 0, +-inf as +-127.  Rows behind the last new one
// keep their bytes.
//
// Bound by memory for a prompt (rows read once from HBM, codes written) and by latency for one token.
#include "kv8.cuh"

namespace mm3fa {

constexpr int KV8_STORE_THREADS = 256;

// N consecutive elements of a row from element e (N * element size a multiple of 16 where vec).
template <int N>
__device__ __forceinline__ void kv8_load(const char * row, int type, int vec, int e, float (&x)[N]) {
    if (type == KV_F32) {
        const float * p = reinterpret_cast<const float *>(row) + e;
        if (vec) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(p + i);
                x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                x[i] = p[i];
            }
        }
        return;
    }
    const uint16_t * p = reinterpret_cast<const uint16_t *>(row) + e;
    uint32_t         w[N / 2];
    if (vec) {
#pragma unroll
        for (int i = 0; i < N / 2; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p + 2 * i);
            w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            w[i] = (uint32_t) p[2 * i] | ((uint32_t) p[2 * i + 1] << 16);
        }
    }
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const float2 f = type == KV_F16 ? h2_to_f2(w[i]) : bf2_to_f2(w[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}

// rne(x / d) clamped to +-127, exactly: q = rint(x * (1/d)) is at most one off next to a tie, and the
// remainder x - q d of an integer quotient next to x / d is exact in F32, so it decides.
__device__ __forceinline__ int kv8_code(float x, float d, float inv) {
    float       q = rintf(x * inv);
    const float r = fmaf(-q, d, x), r2 = 2.0f * fabsf(r);
    if (r2 > d || (r2 == d && (((int) q) & 1))) {
        q += copysignf(1.0f, r);
    }
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    return x != x ? 0 : (int) q;
}

// rne(c * d_old / d) with d_old < d; ratio = d_old / d in F32 puts c * ratio within 127 * 2^-22 of the
// quotient, so only a value that near to a tie needs the 64-bit quotient (c * d_old is exact there).
__device__ __forceinline__ int kv8_requant(int c, float d_old, float d, float ratio) {
    const float t = (float) c * ratio, q = rintf(t);
    if (fabsf(fabsf(t - q) - 0.5f) > 1e-4f) {
        return (int) q;
    }
    return (int) rint((double) c * (double) d_old / (double) d);
}

__global__ void __launch_bounds__(KV8_STORE_THREADS) kv8_append_kernel(const Kv8StoreParams p) {
    constexpr int THREADS = KV8_STORE_THREADS;
    const int     tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int     s = (int) blockIdx.z, h = (int) blockIdx.y >> 1, is_v = (int) blockIdx.y & 1;
    __shared__ float red[THREADS / 32];
    kv8_dep_wait();
    const int P = p.c.P, D = p.c.D;
    const int start = p.start[s];
    const int n     = p.n ? min(max(p.n[s], 0), p.n_rows) : p.n_rows;
    if (start < 0) {
        return;
    }
    const int     j     = (start >> p.c.log2p) + (int) blockIdx.x;  // page slot
    const int64_t first = (int64_t) j << p.c.log2p;                 // its first token
    const int     r0    = max((int) (start - first), 0);            // new rows of the page: [r0, r1)
    const int     r1    = (int) min((int64_t) P, (int64_t) start + n - first);
    const int     page  = kv8_page(p.t, p.c.n_pages, s, j);
    if (page < 0 || r1 <= r0) {
        return;
    }
    const Kv8Rows & x   = is_v ? p.v : p.k;
    const int64_t   ph  = (int64_t) page * p.c.n_head_kv + h;
    int8_t *        dst = (is_v ? p.c.v : p.c.k) + ph * P * D;
    float *         sc  = (is_v ? p.c.v_scale : p.c.k_scale) + ph;
    const char *    src = x.data + (int64_t) h * x.nb2 + (int64_t) s * x.nb3;
    const int       per = D / 16;  // 16-value pieces of a row
    float           amax = 0.0f;
    for (int i = tid; i < (r1 - r0) * per; i += THREADS) {
        float v[16];
        kv8_load<16>(src + (first + r0 + i / per - start) * x.nb1, x.type, x.vec, i % per * 16, v);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float a = fabsf(v[e]);
            amax          = a < INFINITY ? fmaxf(amax, a) : amax;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (lane == 0) {
        red[warp] = amax;
    }
    const float before = r0 > 0 ? *sc : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        amax = fmaxf(amax, red[w]);
    }
    const float d = fmaxf(before, amax / 127.0f);
    if (r0 > 0 && d > before) {
        const float ratio = before / d;
        for (int i = tid; i < r0 * per; i += THREADS) {
            union {
                uint4  u;
                int8_t c[16];
            } w;
            w.u = *reinterpret_cast<const uint4 *>(dst + (int64_t) i * 16);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                w.c[e] = (int8_t) kv8_requant(w.c[e], before, d, ratio);
            }
            *reinterpret_cast<uint4 *>(dst + (int64_t) i * 16) = w.u;
        }
    }
    // a scale whose reciprocal would overflow is brought up by an exact power of two, like its rows
    const float up = d < 1e-30f ? 18446744073709551616.0f : 1.0f, du = d * up;
    const float inv = d > 0.0f ? 1.0f / du : 0.0f;
    for (int i = tid; i < (r1 - r0) * per; i += THREADS) {
        float v[16];
        kv8_load<16>(src + (first + r0 + i / per - start) * x.nb1, x.type, x.vec, i % per * 16, v);
        union {
            uint4  u;
            int8_t c[16];
        } w;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            w.c[e] = (int8_t) (d > 0.0f ? kv8_code(v[e] * up, du, inv) : (v[e] == INFINITY ? 127 : v[e] == -INFINITY ? -127 : 0));
        }
        *reinterpret_cast<uint4 *>(dst + (int64_t) r0 * D + (int64_t) i * 16) = w.u;
    }
    if (tid == 0) {
        *sc = d;
    }
}

// ---- read: rows start[s] .. start[s] + n[s] of each sequence as values; 16 codes per thread
__global__ void __launch_bounds__(KV8_STORE_THREADS) kv8_read_kernel(const Kv8StoreParams p) {
    kv8_dep_wait();
    const int     D = p.c.D, P = p.c.P, per = D / 16;
    const int64_t rows  = (int64_t) p.t.n_seq * p.c.n_head_kv * p.n_rows;
    const int64_t items = 2 * rows * per;
    for (int64_t i = (int64_t) blockIdx.x * KV8_STORE_THREADS + threadIdx.x; i < items;
         i += (int64_t) gridDim.x * KV8_STORE_THREADS) {
        const int     piece = (int) (i % per);
        const int64_t r     = i / per;
        const bool    is_v  = r >= rows;
        const int64_t rr    = is_v ? r - rows : r;
        const int     row   = (int) (rr % p.n_rows);
        const int     h     = (int) (rr / p.n_rows % p.c.n_head_kv);
        const int     s     = (int) (rr / p.n_rows / p.c.n_head_kv);
        const int64_t tok   = (int64_t) p.start[s] + row;
        if (tok < 0 || row >= (p.n ? p.n[s] : p.n_rows) || (tok >> p.c.log2p) >= p.t.max_pages) {
            continue;
        }
        const int page = kv8_page(p.t, p.c.n_pages, s, (int) (tok >> p.c.log2p));
        if (page < 0) {
            continue;
        }
        const int64_t ph = (int64_t) page * p.c.n_head_kv + h;
        const float   sc = (is_v ? p.c.v_scale : p.c.k_scale)[ph];
        union {
            uint4  u;
            int8_t c[16];
        } w;
        w.u = *reinterpret_cast<const uint4 *>((is_v ? p.c.v : p.c.k) + (ph * P + (tok & (P - 1))) * D + piece * 16);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            v[e] = (float) w.c[e] * sc;
        }
        const Kv8Rows & o   = is_v ? p.v : p.k;
        char *          out = o.data + (int64_t) row * o.nb1 + (int64_t) h * o.nb2 + (int64_t) s * o.nb3;
        if (o.type == KV_F32) {
            float * f = reinterpret_cast<float *>(out) + piece * 16;
            if (o.vec) {
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    *reinterpret_cast<float4 *>(f + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    f[e] = v[e];
                }
            }
            continue;
        }
        union {
            uint4    u[2];
            uint16_t h[16];
        } b;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            b.h[e] = o.type == KV_F16 ? __half_as_ushort(__float2half_rn(v[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
        }
        uint16_t * f = reinterpret_cast<uint16_t *>(out) + piece * 16;
        if (o.vec) {
            reinterpret_cast<uint4 *>(f)[0] = b.u[0];
            reinterpret_cast<uint4 *>(f)[1] = b.u[1];
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                f[e] = b.h[e];
            }
        }
    }
}

cudaError_t launch_kv8_append(const Kv8StoreParams & p, cudaStream_t stream) {
    // T rows touch at most ceil((T - 1) / P) + 1 pages of a sequence
    const unsigned pages = (unsigned) ((p.n_rows - 1 + p.c.P - 1) / p.c.P + 1);
    return kv8_launch(kv8_append_kernel, dim3(pages, 2u * (unsigned) p.c.n_head_kv, (unsigned) p.t.n_seq), KV8_STORE_THREADS,
                      0, stream, p);
}

cudaError_t launch_kv8_read(const Kv8StoreParams & p, int sms, cudaStream_t stream) {
    const int64_t items  = 2 * (int64_t) p.t.n_seq * p.c.n_head_kv * p.n_rows * (p.c.D / 16);
    const int64_t blocks = (items + KV8_STORE_THREADS - 1) / KV8_STORE_THREADS;
    return kv8_launch(kv8_read_kernel, dim3((unsigned) (blocks < 8 * sms ? blocks : 8 * sms)), KV8_STORE_THREADS, 0, stream, p);
}

}  // namespace mm3fa
