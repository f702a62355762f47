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
// A page's rows stay in registers between the maximum and the codes, so that they are read once, and the codes
// take no division where a product is sure of them.  Appending 2 prompts of 4096 F32 rows (8 heads, D = 128) and reading
// them back took 60 us with two readings of the rows and a remainder for every code, 53 without the second reading, 38
// so: 20 for the append (84 MB, 63 % of the copy bandwidth of 6.54 TB/s) and 25 for the read (52 %) in graphs of their own.
// The append is bound by issue (slots 68 % busy, DRAM 34 %, 44 % of the warps): the launch bound of 1024 threads holds every
// page size to 64 registers a thread.  The read moves 4 codes a lane and load.  Rows of 16 bits take longer though they are
// half the bytes: 33 us in F16, 36 in BF16.  One token is latency: 6 us for the two.
#include "kv8.cuh"

namespace mm3fa {

constexpr int KS_VALUES = 32;  // of a page's rows that a thread of the append holds: 8 runs of 4
constexpr int KS_READ_THREADS = 256;
constexpr int KS_READ_ROWS    = 64;  // rows per CTA of the read

// 4 consecutive elements of a row from element e (a multiple of 4).
__device__ __forceinline__ void ks_load(const char * row, int type, int vec, int e, float (&x)[4]) {
    if (type == KV_F32) {
        const float * p = reinterpret_cast<const float *>(row) + e;
        if (vec) {
            const float4 f = __ldcs(reinterpret_cast<const float4 *>(p));
            x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = p[i];
            }
        }
        return;
    }
    const uint16_t * p = reinterpret_cast<const uint16_t *>(row) + e;
    uint2            w;
    if (vec) {
        w = __ldcs(reinterpret_cast<const uint2 *>(p));
    } else {
        w.x = (uint32_t) p[0] | ((uint32_t) p[1] << 16), w.y = (uint32_t) p[2] | ((uint32_t) p[3] << 16);
    }
    const float2 a = type == KV_F16 ? h2_to_f2(w.x) : bf2_to_f2(w.x), b = type == KV_F16 ? h2_to_f2(w.y) : bf2_to_f2(w.y);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
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

// P * D / KS_VALUES threads (at least 64)
__global__ void __launch_bounds__(1024) kv8_append_kernel(const Kv8StoreParams p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = (int) blockDim.x;
    const int s = (int) blockIdx.z, h = (int) blockIdx.y >> 1, is_v = (int) blockIdx.y & 1;
    __shared__ float red[32];
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
    const Kv8Rows & x    = is_v ? p.v : p.k;
    const int64_t   ph   = (int64_t) page * p.c.n_head_kv + h;
    int8_t *        dst  = (is_v ? p.c.v : p.c.k) + ph * P * D;
    float *         sc   = (is_v ? p.c.v_scale : p.c.k_scale) + ph;
    const char *    src  = x.data + (int64_t) h * x.nb2 + (int64_t) s * x.nb3 + (first + r0 - start) * x.nb1;
    const int       runs = (r1 - r0) * (D / 4), col = tid % (D / 4), step = threads / (D / 4);  // threads: a multiple of D / 4
    float           v[KS_VALUES / 4][4];
    float           amax = 0.0f;
#pragma unroll
    for (int k = 0; k < KS_VALUES / 4; k++) {
        if (tid + k * threads < runs) {
            ks_load(src + (int64_t) (tid / (D / 4) + k * step) * x.nb1, x.type, x.vec, col * 4, v[k]);
        }
    }
    const float before = r0 > 0 ? *sc : 0.0f;
#pragma unroll
    for (int k = 0; k < KS_VALUES / 4; k++) {
        if (tid + k * threads < runs) {
            amax = fmaxf(fmaxf(amax, fmaxf(fabsf(v[k][0]), fabsf(v[k][1]))), fmaxf(fabsf(v[k][2]), fabsf(v[k][3])));  // not NaN
        }
    }
    if (!(amax < INFINITY)) {  // without infinities
        amax = 0.0f;
#pragma unroll 1
        for (int i = tid; i < runs; i += threads) {
            float y[4];
            ks_load(src + (int64_t) (i / (D / 4)) * x.nb1, x.type, x.vec, col * 4, y);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                amax = fabsf(y[e]) < INFINITY ? fmaxf(amax, fabsf(y[e])) : amax;
            }
        }
    }
    // magnitudes order like their bits
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    if (lane == 0) {
        red[warp] = amax;
    }
    __syncthreads();
    for (int w = 0; w < threads / 32; w++) {
        amax = fmaxf(amax, red[w]);
    }
    const float d = fmaxf(before, amax / 127.0f);
    if (r0 > 0 && d > before) {
        const float ratio = before / d;
        for (int i = tid; i < r0 * (D / 16); i += threads) {
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
#pragma unroll
    for (int k = 0; k < KS_VALUES / 4; k++) {
        if (tid + k * threads < runs) {
            // q = rne(x inv) in the low bits of x inv + 1.5 * 2^23.  x inv is within 127 * 2^-24 of the quotient, so q is
            // right where x inv is 1e-5 away from a tie; the rest (NaN and infinities too) by the remainder
            constexpr float MAGIC = 12582912.0f;
            uint32_t        u[4];
            bool            sure = d >= 1e-30f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float m = fmaf(v[k][e], inv, MAGIC);
                u[e]          = __float_as_uint(m);
                sure          = sure && fabsf(fmaf(v[k][e], inv, MAGIC - m)) <= 0.49999f;
            }
            uint32_t w = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
            if (!sure) {
                w = 0;
#pragma unroll 1
                for (int e = 0; e < 4; e++) {
                    const float a = e == 0 ? v[k][0] : e == 1 ? v[k][1] : e == 2 ? v[k][2] : v[k][3];
                    const int   c = d > 0.0f ? kv8_code(a * up, du, inv) : (a == INFINITY ? 127 : a == -INFINITY ? -127 : 0);
                    w |= (uint32_t) (c & 255) << (8 * e);
                }
            }
            reinterpret_cast<uint32_t *>(dst + (int64_t) r0 * D)[tid + k * threads] = w;
        }
    }
    if (tid == 0) {
        *sc = d;
    }
}

// ---- read: rows start[s] .. start[s] + n[s] of each sequence as values; a warp takes 8 rows, 4 codes a lane at a
// time, so that loads and stores are runs of bytes
template <int D>
__global__ void __launch_bounds__(KS_READ_THREADS) kv8_read_kernel(const Kv8StoreParams p) {
    constexpr int LPR = D / 4, ROWS = KS_READ_ROWS / (KS_READ_THREADS / 32), IT = ROWS * LPR / 32;  // lanes per row, rows per warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = (int) blockIdx.z, h = (int) blockIdx.y >> 1, is_v = (int) blockIdx.y & 1;
    kv8_dep_wait();
    const int       n     = p.n ? min(p.n[s], p.n_rows) : p.n_rows;
    const int64_t   start = p.start[s];
    const Kv8Rows & o     = is_v ? p.v : p.k;
    const int8_t *  pool  = is_v ? p.c.v : p.c.k;
    const float *   scale = is_v ? p.c.v_scale : p.c.k_scale;
    char *          out   = o.data + (int64_t) h * o.nb2 + (int64_t) s * o.nb3;
    const int       r0    = (int) blockIdx.x * KS_READ_ROWS + warp * ROWS;
    // the warp's rows lie in two pages at most (a page has 16 tokens or more)
    const int64_t   tok0 = start + r0;
    const int       in0  = (int) (tok0 & (p.c.P - 1)), split = p.c.P - in0;  // rows of the first page
    const int       j0   = (tok0 >> p.c.log2p) < p.t.max_pages ? (int) (tok0 >> p.c.log2p) : p.t.max_pages;  // negative: kv8_page knows
    const int       pg0  = kv8_page(p.t, p.c.n_pages, s, j0), pg1 = kv8_page(p.t, p.c.n_pages, s, j0 + 1);
    const int64_t   ph0  = (int64_t) max(pg0, 0) * p.c.n_head_kv + h, ph1 = (int64_t) max(pg1, 0) * p.c.n_head_kv + h;
    const float     sc0  = scale[ph0], sc1 = scale[ph1];
    const int8_t *  a0   = pool + (ph0 * p.c.P + in0) * D, *a1 = pool + (ph1 * p.c.P - split) * D;
    uint32_t        w[IT];
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int at = i * 32 + lane, rr = at / LPR;
        w[i] = 0;
        if (r0 + rr < n && tok0 + rr >= 0 && (rr < split ? pg0 : pg1) >= 0) {
            w[i] = *reinterpret_cast<const uint32_t *>((rr < split ? a0 : a1) + at * 4);
        }
    }
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int at = i * 32 + lane, rr = at / LPR, row = r0 + rr, col = at % LPR;
        if (!(row < n && tok0 + rr >= 0 && (rr < split ? pg0 : pg1) >= 0)) {
            continue;
        }
        const float sc = rr < split ? sc0 : sc1;
        float       v[4];
        // 2^23 + (code + 128), exactly, less 2^23 + 128
        const uint32_t u = w[i] ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 | e)) - 8388736.0f) * sc;
        }
        char * dst = out + (int64_t) row * o.nb1;
        if (o.type == KV_F32) {
            float * f = reinterpret_cast<float *>(dst) + col * 4;
            if (o.vec) {
                __stcs(reinterpret_cast<float4 *>(f), make_float4(v[0], v[1], v[2], v[3]));
            } else {
                f[0] = v[0], f[1] = v[1], f[2] = v[2], f[3] = v[3];
            }
            continue;
        }
        uint16_t b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            b[e] = o.type == KV_F16 ? __half_as_ushort(__float2half_rn(v[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
        }
        uint16_t * f = reinterpret_cast<uint16_t *>(dst) + col * 4;
        if (o.vec) {
            __stcs(reinterpret_cast<uint2 *>(f), make_uint2(b[0] | (uint32_t) b[1] << 16, b[2] | (uint32_t) b[3] << 16));
        } else {
            f[0] = b[0], f[1] = b[1], f[2] = b[2], f[3] = b[3];
        }
    }
}

cudaError_t launch_kv8_append(const Kv8StoreParams & p, cudaStream_t stream) {
    // T rows touch at most ceil((T - 1) / P) + 1 pages of a sequence
    const unsigned pages   = (unsigned) ((p.n_rows - 1 + p.c.P - 1) / p.c.P + 1);
    const int      threads = p.c.P * p.c.D / KS_VALUES;
    return kv8_launch(kv8_append_kernel, dim3(pages, 2u * (unsigned) p.c.n_head_kv, (unsigned) p.t.n_seq), threads < 64 ? 64 : threads,
                      0, stream, p);
}

cudaError_t launch_kv8_read(const Kv8StoreParams & p, cudaStream_t stream) {
    const dim3 grid((unsigned) ((p.n_rows + KS_READ_ROWS - 1) / KS_READ_ROWS), 2u * (unsigned) p.c.n_head_kv, (unsigned) p.t.n_seq);
    switch (p.c.D) {
        case 64:
            return kv8_launch(kv8_read_kernel<64>, grid, KS_READ_THREADS, 0, stream, p);
        case 128:
            return kv8_launch(kv8_read_kernel<128>, grid, KS_READ_THREADS, 0, stream, p);
        default:
            return kv8_launch(kv8_read_kernel<256>, grid, KS_READ_THREADS, 0, stream, p);
    }
}

}  // namespace mm3fa
