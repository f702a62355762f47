// kv8_attn.cu - attention over the 8-bit paged KV cache for few query rows (sm_100a): one token or a few
// for each sequence, where the cache has to be streamed once.
//
// Mathematics.  With codes c and page scales a (keys) and b (values), s_j = scale * a * (q . c_j) and
//     o = sum_j 2^(s_j - m) b c_j / sum_j 2^(s_j - m)          (s in log2 units, m a running maximum).
// The codes are exact in F16, so q . c and P . c run on the tensor cores without rounding the cache.
//   * q is brought to [1, 2) at its row's largest element by a power of two (any F32 or BF16 row fits
//     F16 so) and split into an F16 number and the F16 remainder when the result is F32 (25 bits of the
//     row's largest element; one F16 number holds an F16 or BF16 row).
//   * the value scale of a page goes into the weights, P = 2^(s - m) * 2^(m + e - R) * f with b = f 2^e,
//     f in [1, 2), and R the running maximum of (a tile's largest s) + e: O is held in units of 2^R,
//     the sum in units of 2^m, so that pages with scales of any size stay in F16's range.  Weights are
//     rounded to F16 (half a step: 2^-12), and their remainder too when the result is F32.  O, sums
//     and maxima are F32.
//
// Work.  A unit is (sequence, kv head, 16 query rows): rows of all query heads of the group share the
// cache's bytes.  A unit's keys come in blocks of 32; all units' blocks are cut into equal contiguous
// ranges, one per CTA (the lengths are read on the device: a graph replays with others).  In a CTA each of
// the four warps takes every fourth block of a unit through its own ring of cp.async stages - no barrier
// between warps - and keeps its own softmax state; the four are joined in shared memory, and a unit cut
// over CTAs is joined by the last CTA to arrive, in the order of the ranges (no result depends on timing).
#include "kv8.cuh"

namespace mm3fa {

constexpr int KD_WARPS   = 4;
constexpr int KD_THREADS = 32 * KD_WARPS;
constexpr int KD_BLOCK   = 32;     // keys per block
constexpr int KD_ROWS    = 16;     // query rows per unit
constexpr int KD_OFF     = 12;     // P is held times 2^12: F16 keeps 11 bits down to 2^-26 of the largest weight
constexpr int KD_MIN     = 4;      // blocks per CTA below which fewer CTAs take part

template <int D, int NT, bool HP>
struct KdSmem {
    static constexpr int NS    = D == 64 ? (NT == 1 ? 6 : 5) : (D == 128 ? (NT == 1 ? 3 : 2) : 2);  // stages per warp
    static constexpr int TILE  = KD_BLOCK * D;                                    // bytes of K or V
    static constexpr int HEAD  = 32;                                              // scales and flags
    static constexpr int STAGE = 2 * TILE + HEAD;
    static constexpr int RING  = KD_WARPS * NS * STAGE;
    static constexpr int Q     = D / 16 * NT * 32 * (HP ? 16 : 8);  // B fragments
    static constexpr int OROW  = D + 4;                             // floats per row of the merge buffer
    static constexpr int STATE = 2 * NT * 8 * 3 * 4;                // m, l, R
    static constexpr int FIXED = RING + Q + STATE + NT * 8 * 4 + 64;
    static size_t        bytes(int rows) { return FIXED + (size_t) 2 * rows * OROW * 4; }
};

__device__ __forceinline__ uint32_t kd_prmt(uint32_t a, uint32_t b, uint32_t sel) {
    return __byte_perm(a, b, sel);
}

// two codes, offset to 0..255, as F16 values: 0x6400 | u is 1024 + u, exactly
__device__ __forceinline__ uint32_t kd_half2(uint32_t u, uint32_t sel) {
    const uint32_t x    = kd_prmt(u, 0x64646464u, sel);
    const uint32_t bias = 0x64806480u;  // 1152
    const __half2  h    = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void kd_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t kd_movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float kd_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// floor(log2 |x|) within [-126, 126], and 2^e for such e
__device__ __forceinline__ int kd_exponent(float x) {
    return min(max((int) (__float_as_uint(x) >> 23 & 255u) - 127, -126), 126);
}

__device__ __forceinline__ float kd_pow2(int e) {
    return __uint_as_float((uint32_t) (e + 127) << 23);
}

__device__ __forceinline__ void kd_cp16(uint32_t dst, const void * src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void kd_cp4(uint32_t dst, const void * src, uint32_t n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ uint32_t kd_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 16-byte chunk c of a tile's row r is kept at chunk c ^ swz(r): the K and V fragment loads (8 lanes of two
// rows and four column groups, or of four rows and two) then touch each bank once.  D = 64 has two rows
// in 128 bytes.
template <int D>
__device__ __forceinline__ int kd_swz(int r) {
    return D == 64 ? (r >> 1) & 3 : r & 7;
}

struct KdSeq {
    int n;   // keys
    int m;   // query rows (positions)
    int nb;  // blocks of keys, at least one: a unit without keys still writes its zeros
};

__device__ __forceinline__ KdSeq kd_seq(const Kv8AttnParams & p, int s) {
    KdSeq q;
    q.n  = min(max(p.kv_len[s], 0), p.t.max_pages * p.c.P);
    q.m  = p.q_len ? min(max(p.q_len[s], 0), p.n_q) : p.n_q;
    q.n  = q.m ? q.n : 0;
    q.nb = max(1, (q.n + KD_BLOCK - 1) / KD_BLOCK);
    return q;
}

// A walk over the segments (unit, blocks [b, e)) of a CTA's range.
struct KdWalk {
    int     s, u;  // sequence, unit of it
    int     b, e;
    int64_t left;  // blocks from b on
    KdSeq   q;
    __device__ __forceinline__ void open(const Kv8AttnParams & p) {
        q = kd_seq(p, s);
        e = (int) min((int64_t) q.nb, b + left);
    }
    // to the next segment; false at the end of the range
    __device__ __forceinline__ bool next(const Kv8AttnParams & p, int units) {
        left -= e - b;
        if (left <= 0) {
            return false;
        }
        b = 0;
        if (++u == units) {
            u = 0;
            s++;
            q = kd_seq(p, s);
        }
        e = (int) min((int64_t) q.nb, left);
        return true;
    }
};

template <int D, int NT, bool HP>
__global__ void __launch_bounds__(KD_THREADS) kv8_decode_kernel(const Kv8AttnParams p) {
    using L          = KdSmem<D, NT, HP>;
    constexpr int NS = L::NS, CH = D / 64, MT = D / 16;
    extern __shared__ __align__(16) char smem[];
    __shared__ int64_t sh_total;
    __shared__ int64_t sh_scan[KD_WARPS];
    __shared__ int     sh_s, sh_u, sh_b, sh_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    char *    ring   = smem + warp * NS * L::STAGE;
    char *    qf     = smem + L::RING;
    float *   state  = reinterpret_cast<float *>(qf + L::Q);          // [2][row][m, l, R]
    float *   qscale = state + 2 * NT * 8 * 3;                        // [row]
    float *   obuf   = reinterpret_cast<float *>(smem + L::FIXED);    // [2][row][OROW]
    const int all_rows = p.ratio * p.n_q, groups = (all_rows + KD_ROWS - 1) / KD_ROWS;
    const int units = p.c.n_head_kv * groups;  // of a sequence
    kv8_dep_wait();

    // ---- this CTA's range of blocks: the sequences' block counts, scanned
    int64_t   sum = 0;
    const int per = (p.t.n_seq + KD_THREADS - 1) / KD_THREADS, s0 = min(tid * per, p.t.n_seq), s1 = min(s0 + per, p.t.n_seq);
    for (int s = s0; s < s1; s++) {
        sum += (int64_t) kd_seq(p, s).nb * units;
    }
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        inc += lane >= o ? x : 0;
    }
    if (lane == 31) {
        sh_scan[warp] = inc;
    }
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < KD_WARPS; w++) {
        inc += w < warp ? sh_scan[w] : 0;
        total += sh_scan[w];
    }
    const int64_t ctas = min((int64_t) gridDim.x, (total + KD_MIN - 1) / KD_MIN);
    const int64_t c    = blockIdx.x;
    if (c >= ctas) {
        return;
    }
    const int64_t begin = c * total / ctas, end = (c + 1) * total / ctas;
    if (inc - sum <= begin && begin < inc) {  // the one thread whose sequences hold the first block
        int64_t off = begin - (inc - sum);
        int     s   = s0, nb = kd_seq(p, s).nb;
        while (off >= (int64_t) nb * units) {
            off -= (int64_t) nb * units;
            nb = kd_seq(p, ++s).nb;
        }
        sh_s = s, sh_u = (int) (off / nb), sh_b = (int) (off % nb);
        sh_total = begin - off;  // first block of sequence s
    }
    __syncthreads();
    KdWalk seg;
    seg.s = sh_s, seg.u = sh_u, seg.b = sh_b, seg.left = end - begin;
    int64_t seq_first = sh_total;
    seg.open(p);

    // ---- the warp's loads: block after block of the same walk, NS - 1 stages ahead
    KdWalk ld     = seg;
    int    ld_b   = ld.b + warp;
    bool   ld_on  = true;
    int    pg0 = -1, pg1 = -1;  // pages of the next block's halves
    auto   settle = [&] {       // brings the load cursor to a block of this warp and reads its pages
        while (ld_on && ld_b >= ld.e) {
            ld_on = ld.next(p, units);
            ld_b  = ld.b + warp;
        }
        if (ld_on) {
            const int k0 = ld_b * KD_BLOCK, j = k0 >> p.c.log2p;
            pg0 = k0 < ld.q.n ? kv8_page(p.t, p.c.n_pages, ld.s, j) : -1;
            pg1 = p.c.log2p > 4 ? pg0 : (k0 + 16 < ld.q.n ? kv8_page(p.t, p.c.n_pages, ld.s, j + 1) : -1);
        }
    };
    int  ld_stage = 0;
    auto load     = [&] {
        if (ld_on) {
            char *         st  = ring + ld_stage * L::STAGE;
            const int      h   = ld.u / groups;
            const int      row = (ld_b * KD_BLOCK) & (p.c.P - 1);  // of the block in its page
            const int64_t  ph0 = (int64_t) max(pg0, 0) * p.c.n_head_kv + h, ph1 = (int64_t) max(pg1, 0) * p.c.n_head_kv + h;
            const int64_t  o0 = (ph0 * p.c.P + row) * D;
            const int64_t  o1 = (p.c.log2p > 4 ? o0 + 16 * D : ph1 * p.c.P * D);
            const uint32_t z0 = pg0 >= 0 ? 16u : 0u, z1 = pg1 >= 0 ? 16u : 0u;
            const uint32_t dst = smem_addr(st);
#pragma unroll
            for (int i = 0; i < 4 * CH; i++) {  // 32 rows of D / 16 chunks, 32 chunks at a time
                const int     idx  = i * 32 + lane, r = idx / (D / 16), ck = idx % (D / 16);
                const bool    half = i >= 2 * CH;
                const int64_t off  = (half ? o1 - 16 * D : o0) + (int64_t) idx * 16;
                const uint32_t to  = dst + (uint32_t) (r * D + ((ck ^ kd_swz<D>(r)) << 4));
                kd_cp16(to, p.c.k + off, half ? z1 : z0);
                kd_cp16(to + L::TILE, p.c.v + off, half ? z1 : z0);
            }
            if (lane < 4) {
                const int64_t ph = lane & 1 ? ph1 : ph0;
                kd_cp4(dst + 2 * L::TILE + lane * 4, (lane < 2 ? p.c.k_scale : p.c.v_scale) + ph, (lane & 1 ? z1 : z0) / 4);
            } else if (lane < 6) {
                reinterpret_cast<int *>(st + 2 * L::TILE)[lane] = (lane & 1 ? pg1 : pg0) >= 0;
            }
            ld_b += KD_WARPS;
            settle();
        }
        ld_stage = ld_stage + 1 == NS ? 0 : ld_stage + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    settle();
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
        load();
    }
    int stage = 0;

    for (bool more = true; more;) {
        const int  h = seg.u / groups, r0 = (seg.u % groups) * KD_ROWS;
        const int  rows  = min(all_rows - r0, min(KD_ROWS, NT * 8));
        const KdSeq sq   = seg.q;
        const int   low  = p.causal ? max(sq.n - (sq.m - 1), 0) : sq.n;  // keys below this are seen by every row
        // ---- Q fragments: for k-step i, column n, lane (g = n, t): the dims of chunk list(t), bytes 4i .. 4i + 3
        for (int rr = warp; rr < NT * 8; rr += KD_WARPS) {
            constexpr int E = D / 32;
            float         x[E], amax = 0.0f;
            const int     r = r0 + rr, qi = r / p.ratio, hq = h * p.ratio + r % p.ratio;
            const bool    live = rr < rows && qi < sq.m;
            if (live) {
                const char * src = p.q.data + (int64_t) qi * p.q.nb1 + (int64_t) hq * p.q.nb2 + (int64_t) seg.s * p.q.nb3;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int i = lane * E + e;
                    x[e]        = p.q.type == KV_F32 ? reinterpret_cast<const float *>(src)[i]
                                : p.q.type == KV_F16 ? __half2float(reinterpret_cast<const __half *>(src)[i])
                                                     : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(src)[i]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    x[e] = 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                amax = fmaxf(amax, fabsf(x[e]));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            }
            // exponent of the row's largest element; rows of zeros, infinities and NaN stay as they are
            const int   ex = amax > 0.0f && amax < INFINITY ? kd_exponent(amax) : 0;
            const float dn = kd_pow2(-ex);
            if (lane == 0) {
                qscale[rr] = kd_pow2(ex) * p.scale * (p.softcap > 0.0f ? 1.0f / p.softcap : LOG2E);
            }
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const int      d   = lane * E + e;  // even; its pair sits in one fragment register
                const int      ck  = d >> 4, by = d & 15;
                const int      tt  = D == 64 ? ck : (ck & 7) >> 1;
                const int      jj  = D == 64 ? 0 : (ck & 1) + 2 * (ck >> 3);
                const int      ks  = jj * 4 + (by >> 2), hi = (by >> 1) & 1;
                const float    a = x[e] * dn, b = x[e + 1] * dn;
                const __half2  w  = __floats2half2_rn(a, b);
                uint32_t *     to = reinterpret_cast<uint32_t *>(qf) + ((ks * NT + (rr >> 3)) * 32 + (rr & 7) * 4 + tt) * (HP ? 4 : 2) + hi;
                to[0]             = *reinterpret_cast<const uint32_t *>(&w);
                if (HP) {
                    const float2 f = __half22float2(w);
                    to[2]          = kd_pack(a - f.x, b - f.y);
                }
            }
        }
        __syncthreads();
        float qs[NT][2], m[NT][2], l[NT][2], R[NT][2], o[MT][NT][4];
        int   lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int rr = nt * 8 + 2 * t + i, qi = (r0 + rr) / p.ratio;
                qs[nt][i]  = qscale[rr];
                lim[nt][i] = p.causal ? sq.n - (sq.m - 1 - qi) : sq.n;
                m[nt][i] = -INFINITY, l[nt][i] = 0.0f, R[nt][i] = -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
            }
        }

        for (int b = seg.b + warp; b < seg.e; b += KD_WARPS) {
            asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
            __syncwarp();
            load();  // into the stage that the last block has left
            const char *   st   = ring + stage * L::STAGE;
            const float4   sc   = *reinterpret_cast<const float4 *>(st + 2 * L::TILE);  // a0, a1, b0, b1
            const int2     has  = *reinterpret_cast<const int2 *>(st + 2 * L::TILE + 16);
            float          s[2][NT][4];
#pragma unroll
            for (int a = 0; a < 2; a++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s[a][nt][0] = s[a][nt][1] = s[a][nt][2] = s[a][nt][3] = 0.0f;
                }
            }
            // S^T = K Q^T: keys 16a + g and 16a + g + 8 of lane g, in the chunks of lane t
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const int ck = D == 64 ? t : 2 * t + (j & 1) + 8 * (j >> 1);
                uint4     w[2][2];
#pragma unroll
                for (int a = 0; a < 2; a++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int r = 16 * a + 8 * i + g;
                        w[a][i]     = *reinterpret_cast<const uint4 *>(st + r * D + ((ck ^ kd_swz<D>(r)) << 4));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t bq[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const char * f = qf + (((j * 4 + i) * NT + nt) * 32 + lane) * (HP ? 16 : 8);
                        if (HP) {
                            const uint4 u = *reinterpret_cast<const uint4 *>(f);
                            bq[nt][0] = u.x, bq[nt][1] = u.y, bq[nt][2] = u.z, bq[nt][3] = u.w;
                        } else {
                            const uint2 u = *reinterpret_cast<const uint2 *>(f);
                            bq[nt][0] = u.x, bq[nt][1] = u.y;
                        }
                    }
#pragma unroll
                    for (int a = 0; a < 2; a++) {
                        const uint32_t x = (&w[a][0].x)[i] ^ 0x80808080u, y = (&w[a][1].x)[i] ^ 0x80808080u;
                        const uint32_t f[4] = { kd_half2(x, 0x4140), kd_half2(y, 0x4140), kd_half2(x, 0x4342), kd_half2(y, 0x4342) };
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            kd_mma(s[a][nt], f, bq[nt][0], bq[nt][1]);
                            if (HP) {
                                kd_mma(s[a][nt], f, bq[nt][2], bq[nt][3]);
                            }
                        }
                    }
                }
            }
            // scores in log2 units; -inf for keys that a row does not see
            const int  k0   = b * KD_BLOCK;
            const bool part = k0 + KD_BLOCK > low || !(has.x & has.y);
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const float as = a ? sc.y : sc.x;
                const bool  ok = (a ? has.y : has.x) != 0;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = s[a][nt][e] * (qs[nt][e & 1] * as);
                        if (p.softcap > 0.0f) {
                            x = p.softcap * LOG2E * tanhf(x);
                        }
                        if (part) {
                            const int key = k0 + 16 * a + g + 8 * (e >> 1);
                            x             = ok && key < lim[nt][e & 1] ? x : -INFINITY;
                        }
                        s[a][nt][e] = x;
                    }
                }
            }
            // value scales: b = vf * 2^ve, vf in [1, 2); 0 where a page has none
            int   ve[2];
            float vf[2];
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const float v = a ? sc.w : sc.z;
                ve[a]         = kd_exponent(v);
                vf[a]         = v * kd_pow2(-ve[a]);
            }
            uint32_t ph[2][NT][2], pl[2][NT][2];
            float    grow[NT][2];
            bool     up = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    // the row's largest score of each half; one value where the halves share a page
                    float t0 = fmaxf(s[0][nt][i], s[0][nt][i + 2]), t1 = fmaxf(s[1][nt][i], s[1][nt][i + 2]);
                    if (p.c.log2p > 4) {
                        t0 = fmaxf(t0, t1);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
                    }
                    if (p.c.log2p > 4) {
                        t1 = t0;
                    } else {
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) {
                            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
                        }
                    }
                    const float mn = fmaxf(m[nt][i], fmaxf(t0, t1));
                    const float ms = mn == -INFINITY ? 0.0f : mn;  // no key yet: every weight is 2^-inf
                    float       rn = R[nt][i];
                    rn = sc.z != 0.0f ? fmaxf(rn, t0 + (float) ve[0]) : rn;
                    rn = sc.w != 0.0f ? fmaxf(rn, t1 + (float) ve[1]) : rn;
                    const float rs = rn == -INFINITY ? 0.0f : rn;
                    l[nt][i] *= kd_ex2(m[nt][i] - ms);
                    grow[nt][i] = kd_ex2(R[nt][i] - rs);
                    up |= rn > R[nt][i];
                    m[nt][i] = mn, R[nt][i] = rn;
#pragma unroll
                    for (int a = 0; a < 2; a++) {
                        // capped where the largest score is so far above that the weights are 0 anyway
                        const float f = (a ? sc.w : sc.z) != 0.0f ? kd_ex2(fminf(ms + (float) ve[a] - rs + KD_OFF, 120.0f)) * vf[a] : 0.0f;
#pragma unroll
                        for (int e = i; e < 4; e += 2) {
                            const float w  = kd_ex2(s[a][nt][e] - ms);
                            l[nt][i]      += w;
                            s[a][nt][e]    = w * f;
                        }
                    }
                }
#pragma unroll
                for (int a = 0; a < 2; a++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t hi = kd_pack(s[a][nt][2 * k], s[a][nt][2 * k + 1]);
                        ph[a][nt][k]      = kd_movmatrix(hi);
                        if (HP) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                            pl[a][nt][k]   = kd_movmatrix(kd_pack(s[a][nt][2 * k] - f.x, s[a][nt][2 * k + 1] - f.y));
                        }
                    }
                }
            }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        o[i][nt][0] *= grow[nt][0], o[i][nt][1] *= grow[nt][1];
                        o[i][nt][2] *= grow[nt][0], o[i][nt][3] *= grow[nt][1];
                    }
                }
            }
            // O^T += V^T P^T: dims of chunk g (two per row pair of an MMA), keys 2t, 2t + 1, 2t + 8, 2t + 9
            const char * vt = st + L::TILE;
#pragma unroll
            for (int a = 0; a < 2; a++) {
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; j++) {
                    constexpr int WORDS = D == 64 ? 2 : 4;
                    uint32_t      w[4][WORDS];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 16 * a + 2 * t + (i & 1) + 8 * (i >> 1);
                        if (D == 64) {
                            const uint2 u = *reinterpret_cast<const uint2 *>(vt + r * D + (((g >> 1) ^ kd_swz<D>(r)) << 4) + (g & 1) * 8);
                            w[i][0] = u.x, w[i][1] = u.y;
                        } else {
                            const uint4 u = *reinterpret_cast<const uint4 *>(vt + r * D + (((g + 8 * j) ^ kd_swz<D>(r)) << 4));
                            w[i][0] = u.x, w[i][1] = u.y, w[i][WORDS - 2] = u.z, w[i][WORDS - 1] = u.w;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < WORDS; k++) {
                        const uint32_t x0 = w[0][k] ^ 0x80808080u, x1 = w[1][k] ^ 0x80808080u;
                        const uint32_t x2 = w[2][k] ^ 0x80808080u, x3 = w[3][k] ^ 0x80808080u;
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const uint32_t y = kd_prmt(x0, x1, q ? 0x7362 : 0x5140), z = kd_prmt(x2, x3, q ? 0x7362 : 0x5140);
                            const uint32_t f[4] = { kd_half2(y, 0x4140), kd_half2(y, 0x4342), kd_half2(z, 0x4140), kd_half2(z, 0x4342) };
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                kd_mma(o[j * 8 + 2 * k + q][nt], f, ph[a][nt][0], ph[a][nt][1]);
                                if (HP) {
                                    kd_mma(o[j * 8 + 2 * k + q][nt], f, pl[a][nt][0], pl[a][nt][1]);
                                }
                            }
                        }
                    }
                }
            }
            stage = stage + 1 == NS ? 0 : stage + 1;
        }

        // ---- the four warps' states, joined: warps 2 and 3 into 0 and 1 (each lane at its own place), then those
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
                }
            }
        }
#pragma unroll
        for (int round = 0; round < 2; round++) {
            if (round == 1) {
                __syncthreads();
            }
            if (round == 0 ? warp >= 2 : warp < 2) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int rr = nt * 8 + 2 * t + i;
                        float *   st = state + ((warp & 1) * NT * 8 + rr) * 3;
                        float *   w  = obuf + ((warp & 1) * rows + rr) * L::OROW;
                        float     fa = 1.0f, fb = 0.0f;
                        if (round == 1) {
                            const float mb = st[0], lb = st[1], Rb = st[2];
                            const float mn = fmaxf(m[nt][i], mb), rn = fmaxf(R[nt][i], Rb);
                            const float ms = mn == -INFINITY ? 0.0f : mn, rs = rn == -INFINITY ? 0.0f : rn;
                            l[nt][i] = l[nt][i] * kd_ex2(m[nt][i] - ms) + lb * kd_ex2(mb - ms);
                            fa = kd_ex2(R[nt][i] - rs), fb = kd_ex2(Rb - rs);
                            m[nt][i] = mn, R[nt][i] = rn;
                            __syncwarp();
                        }
                        if (g == 0) {
                            st[0] = m[nt][i], st[1] = l[nt][i], st[2] = R[nt][i];
                        }
                        if (rr < rows) {
#pragma unroll
                            for (int j = 0; j < MT / 2; j++) {
                                // 4 dims at a time, rotated by t: no bank twice
                                const int jj = MT / 2 < 4 ? (j + t) & 1 : (j & ~3) | ((j + t) & 3);
                                const int d  = D == 64 ? 8 * g + 4 * jj : (jj >> 2) * 128 + 16 * g + 4 * (jj & 3);
                                float4    v  = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                                for (int k = 0; k < MT / 2; k++) {
                                    if (k == jj) {
                                        v = make_float4(o[2 * k][nt][i], o[2 * k][nt][i + 2], o[2 * k + 1][nt][i], o[2 * k + 1][nt][i + 2]);
                                    }
                                }
                                if (round == 1) {
                                    const float4 y = *reinterpret_cast<const float4 *>(w + d);
                                    v.x = v.x * fa + y.x * fb, v.y = v.y * fa + y.y * fb;
                                    v.z = v.z * fa + y.z * fb, v.w = v.w * fa + y.w * fb;
                                }
                                *reinterpret_cast<float4 *>(w + d) = v;
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
        const int64_t first = seq_first + (int64_t) seg.u * sq.nb;  // the unit's first block
        const bool    whole = seg.b == 0 && seg.e == sq.nb;
        float *       slot  = p.part + (2 * c + (seg.b == 0)) * (int64_t) KD_ROWS * (D + 4);
        // O (in units of 2^(R - KD_OFF)) over the sum (of 2^m); rows without keys, and without a value scale, are 0
        auto write = [&](int rr, int d, float4 v, float mt, float lt, float rt) {
            const int r = r0 + rr, qi = r / p.ratio, hq = h * p.ratio + r % p.ratio;
            if (qi >= sq.m) {
                return;
            }
            const float inv = lt != 0.0f ? (1.0f / (1 << KD_OFF)) / lt : 0.0f, up = rt == -INFINITY ? 0.0f : kd_ex2(rt - mt);
            v.x = v.x * inv * up, v.y = v.y * inv * up, v.z = v.z * inv * up, v.w = v.w * inv * up;
            char * dst = p.o.data + (int64_t) hq * p.o.nb1 + (int64_t) qi * p.o.nb2 + (int64_t) seg.s * p.o.nb3;
            if (p.o.type == KV_F32) {
                float * f = reinterpret_cast<float *>(dst) + d;
                if (p.o.vec) {
                    *reinterpret_cast<float4 *>(f) = v;
                } else {
                    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
                }
                return;
            }
            uint16_t * f = reinterpret_cast<uint16_t *>(dst) + d;
            const float x[4] = { v.x, v.y, v.z, v.w };
            uint16_t    y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                y[e] = p.o.type == KV_F16 ? __half_as_ushort(__float2half_rn(x[e])) : __bfloat16_as_ushort(__float2bfloat16_rn(x[e]));
            }
            if (p.o.vec) {
                *reinterpret_cast<uint2 *>(f) = make_uint2(y[0] | (uint32_t) y[1] << 16, y[2] | (uint32_t) y[3] << 16);
            } else {
                f[0] = y[0], f[1] = y[1], f[2] = y[2], f[3] = y[3];
            }
        };
        for (int it = tid; it < rows * (D / 4); it += KD_THREADS) {
            const int rr = it / (D / 4), d = it % (D / 4) * 4;
            float     mt = -INFINITY, rt = -INFINITY, lt = 0.0f;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const float * x = state + (w * NT * 8 + rr) * 3;
                mt = fmaxf(mt, x[0]), rt = fmaxf(rt, x[2]);
            }
            const float ms = mt == -INFINITY ? 0.0f : mt, rs = rt == -INFINITY ? 0.0f : rt;
            float4      v  = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const float * x = state + (w * NT * 8 + rr) * 3;
                const float   f = kd_ex2(x[2] - rs);
                const float4  y = *reinterpret_cast<const float4 *>(obuf + (w * rows + rr) * L::OROW + d);
                lt += x[1] * kd_ex2(x[0] - ms);
                v.x += y.x * f, v.y += y.y * f, v.z += y.z * f, v.w += y.w * f;
            }
            if (whole) {
                write(rr, d, v, mt, lt, rt);
            } else {
                *reinterpret_cast<float4 *>(slot + rr * (D + 4) + d) = v;
                if (d == 0) {
                    *reinterpret_cast<float4 *>(slot + rr * (D + 4) + D) = make_float4(mt, lt, rt, 0.0f);
                }
            }
        }
        if (!whole) {
            // the CTAs that hold a part of the unit: range k is [k total / ctas, (k + 1) total / ctas)
            const int64_t c0 = ((first + 1) * ctas - 1) / total, c1 = ((first + sq.nb) * ctas - 1) / total;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t seen = atomicAdd(&p.counters[c0], 1u);
                sh_last             = seen == (uint32_t) (c1 - c0);
                if (sh_last) {
                    p.counters[c0] = 0;
                }
            }
            __syncthreads();
            if (sh_last) {
                __threadfence();
                for (int it = tid; it < rows * (D / 4); it += KD_THREADS) {
                    const int rr = it / (D / 4), d = it % (D / 4) * 4;
                    float     mt = -INFINITY, rt = -INFINITY, lt = 0.0f;
                    float4    v  = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int64_t k = c0; k <= c1; k++) {
                        const float * x = p.part + (2 * k + (k == c0)) * (int64_t) KD_ROWS * (D + 4) + rr * (D + 4);
                        const float4  y = __ldcg(reinterpret_cast<const float4 *>(x + d));
                        const float4  z = __ldcg(reinterpret_cast<const float4 *>(x + D));
                        const float   mn = fmaxf(mt, z.x), rn = fmaxf(rt, z.z);
                        const float   ms = mn == -INFINITY ? 0.0f : mn, rs = rn == -INFINITY ? 0.0f : rn;
                        const float   f = kd_ex2(rt - rs), e = kd_ex2(z.z - rs);
                        lt  = lt * kd_ex2(mt - ms) + z.y * kd_ex2(z.x - ms);
                        v.x = v.x * f + y.x * e, v.y = v.y * f + y.y * e, v.z = v.z * f + y.z * e, v.w = v.w * f + y.w * e;
                        mt = mn, rt = rn;
                    }
                    write(rr, d, v, mt, lt, rt);
                }
            }
        }
        const int s_before = seg.s;
        more               = seg.next(p, units);
        if (more && seg.s != s_before) {
            seq_first += (int64_t) sq.nb * units;
        }
        __syncthreads();  // state, obuf and the Q fragments are written again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

namespace {

template <int D, int NT, bool HP>
cudaError_t launch_one(const Kv8AttnParams & p, unsigned ctas, int rows, cudaStream_t stream) {
    const size_t smem = KdSmem<D, NT, HP>::bytes(rows);
    // per device, so that a second device gets it too; cheap
    const cudaError_t e = cudaFuncSetAttribute(kv8_decode_kernel<D, NT, HP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int) KdSmem<D, NT, HP>::bytes(NT * 8));
    return e != cudaSuccess ? e : kv8_launch(kv8_decode_kernel<D, NT, HP>, dim3(ctas), KD_THREADS, smem, stream, p);
}

template <int D>
cudaError_t launch_d(const Kv8AttnParams & p, unsigned ctas, int rows, bool hp, cudaStream_t stream) {
    if (rows <= 8) {
        return hp ? launch_one<D, 1, true>(p, ctas, rows, stream) : launch_one<D, 1, false>(p, ctas, rows, stream);
    }
    return hp ? launch_one<D, 2, true>(p, ctas, rows, stream) : launch_one<D, 2, false>(p, ctas, rows, stream);
}

// CTAs that an SM holds at once: two, by shared memory, but for D = 256
int ctas_per_sm(int D) {
    return D == 256 ? 1 : 2;
}

}  // namespace

// Counters (one per CTA) and two partial results per CTA, whatever the lengths are.
size_t kv8_attn_workspace_bytes(int D, int n_q, int ratio, int n_head_kv, int n_seq, int sms) {
    const size_t ctas = (size_t) sms * (size_t) ctas_per_sm(D);
    (void) n_q, (void) ratio, (void) n_head_kv, (void) n_seq;
    return WS_STATUS_BYTES + (ctas * 4 + 255) / 256 * 256 + 2 * ctas * KD_ROWS * (size_t) (D + 4) * 4;
}

cudaError_t launch_kv8_attn(const Kv8AttnParams & p0, int sms, cudaStream_t stream) {
    Kv8AttnParams p    = p0;
    const int     most = sms * ctas_per_sm(p.c.D);
    p.counters = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(p.status) + WS_STATUS_BYTES);
    p.part     = reinterpret_cast<float *>(reinterpret_cast<char *>(p.counters) + ((size_t) most * 4 + 255) / 256 * 256);
    const int     all = p.ratio * p.n_q, rows = all < KD_ROWS ? all : KD_ROWS;
    const int64_t units  = (int64_t) p.t.n_seq * p.c.n_head_kv * ((all + KD_ROWS - 1) / KD_ROWS);
    const int64_t blocks = units * (((int64_t) p.t.max_pages * p.c.P + KD_BLOCK - 1) / KD_BLOCK);  // at most
    const int64_t want   = (blocks + KD_MIN - 1) / KD_MIN;
    const unsigned ctas  = (unsigned) (want < most ? want : most);
    const bool     hp    = p.o.type == KV_F32;
    switch (p.c.D) {
        case 64:
            return launch_d<64>(p, ctas, rows, hp, stream);
        case 128:
            return launch_d<128>(p, ctas, rows, hp, stream);
        default:
            return launch_d<256>(p, ctas, rows, hp, stream);
    }
}

}  // namespace mm3fa
