// kv8_attn.cu - attention over the 8-bit paged KV cache for few query rows (sm_100a): one token or a few
// for each sequence, where the cache has to be streamed once.
//
// Mathematics.  With codes c and page scales a (keys) and b (values), s_j = scale * a * (q . c_j) and
//     o = sum_j 2^(s_j - m) b c_j / sum_j 2^(s_j - m)          (s in log2 units, m a running maximum).
//   * q . c in integers: a row of q becomes fixed-point numbers of four 8-bit digits, the largest element in
//     [2^29, 2^30), and each digit's dot with the codes is exact on the 8-bit tensor cores.  No element is off by more
//     than 2^-30 of the row's largest; F32 ones down to 2^-6 of it, F16 ones to 2^-19 and BF16 ones to 2^-22 are exact.
//     (With three digits for F32 and two for 16-bit results the small elements beside a large one decided wrongly: one of
//     1000 among N(0, 1), with keys of 0 there, put F16 results 5 half steps off.  48 sequences of up to 10240 tokens
//     took 105 us in BF16 so, 115 now; F32 118 and 120.)
//   * P . c in F16, which holds the codes exactly.  The value scale of a page goes into the weights,
//     P = 2^(s - m) * 2^(m + e - R) * f with b = f 2^e, f in [1, 2), and R the running maximum of (a tile's
//     largest s) + e: O is held in units of 2^R, the sum in units of 2^m, so that pages with scales of
//     any size stay in F16's range.  Weights are rounded to F16 (half a step: 2^-12), which
//     is below what a BF16 result keeps; for F32 and F16 results their remainder is a second operand.  O, sums and maxima are F32.
//     The tensor core truncates what it adds to an F32 accumulator, always towards zero: 4e-10 of the result a key (3.4e-6
//     over 8000).  For an F32 result, and for 16-bit ones of tables over KD_LONG tokens, it sums the keys of a block from 0, and
//     O takes the sums by additions that round (1e-7 over 8000; 48 sequences of up to 10240, F32: 123 us against 120).
//
// Work.  A unit is (sequence, kv head, 16 query rows): rows of all query heads of the group share the
// cache's bytes.  A unit's keys come in blocks of 32.  Every CTA finds its work from the lengths on the
// device (a graph replays with others), by one of three cuts:
//   whole  no unit above KD_WHOLE blocks, or units so much alike that no cut is worth a crossing: whole units, an
//          equal number for each CTA;
//   split  few units: each in parts of up to W blocks, one part per CTA, W so that all parts run at once;
//   flat   otherwise: all units' blocks in a row, in equal contiguous ranges, one per CTA.
// Flat ranges are even, but a CTA that crosses from one unit to the next pays a second start and end, about
// KD_CROSS blocks of its time; parts are uneven by the last part of each unit: total / (G - U) against
// total / G blocks for the longest of G CTAs with U units.
// In a CTA each of the four warps takes every fourth block of a unit through its own ring of cp.async
// stages - no barrier between warps - and keeps its own softmax state; the four are joined in shared
// memory, and the parts of a unit by the last CTA to arrive, in their order (no result depends on timing).
//
// Bound.  One token of 48 sequences of 1 to 10240 tokens (32 heads on 8, D = 128, BF16): 115 us in a graph, 67 % of the copy
// bandwidth of 6.54 TB/s (125 us for a call by itself); issue slots are half busy and DRAM half, each of an SM's 12 warps
// waiting for its own next block.  110 of 2000 each: 93 us and 75 %.  For two of 8192 (F32: 19.8 us, 33.6 MB, floor 5.1 us; 19.5
// where 36 layers' caches are read in turn) the start - lengths, table, first pages, one after another - and the join of the
// parts through global memory are most of the 9.6 us that a call over a hundred tokens takes, and the 9 blocks of a CTA, 2 or 3
// a warp, end before the rings reach their rate: the decode over an F16 slab, which joins in clusters, takes 14.4 there.  From
// 9 rows on (NT = 2) it is issue: 0.9 us for a block of a CTA, two CTAs an SM (16 sequences of 1024, 64 rows per kv head:
// 58 us).  Two stages for three CTAs of an SM against three stages for two, D = 128, one row per head:
// 115 us against 130 for the 48 sequences, 20.8 against 19.2 for the two.
#include "kv8.cuh"
#include "tc_sm100.cuh"

#include <algorithm>

namespace mm3fa {

constexpr int KD_WARPS   = 4;
constexpr int KD_THREADS = 32 * KD_WARPS;
constexpr int KD_BLOCK   = 32;     // keys per block
constexpr int KD_ROWS    = 16;     // query rows per unit
constexpr int KD_OFF     = 12;     // P is held times 2^12: F16 keeps 11 bits down to 2^-26 of the largest weight
// 2 sequences of 300: 10.4 us whole, 9.6 in parts (F32; BF16 10.0 and 9.8); 100 of 400 (BF16): 29.3 whole, 35.9 flat.
constexpr int KD_WHOLE   = 16;
// Blocks of a part, at least: 4, 8, 16 take 11.8, 11.8, 14.8 us for one sequence of 2000.
constexpr int KD_PART    = 4;
// What a crossing costs, in blocks.  0, 8, 32: 25.5, 20.1, 20.7 us for 2 sequences of 8192 (0: flat), 40.2, 39.9, 39.1
// for 16 of 4096 (32: parts).  Whole against flat: 29.5 against 35.7 us for 50 of 1000, 92.7 against 101.3 for 110 of 2000.
constexpr int KD_CROSS   = 32;

// Tokens up to which sums in the tensor core's truncating accumulators (4e-10 of the result a key) stay an eighth of F16's
// half step.
constexpr int KD_LONG    = 65536;

constexpr int KD_SM_BYTES  = 228 * 1024;  // shared memory of an SM
constexpr int KD_CTA_BYTES = 1024;        // what each CTA on it takes beside its own

template <int D, int NT>
struct KdSmem {
    // CTAs per SM and stages per warp: what shared memory and registers hold
    static constexpr int CTAS  = D == 64 ? (NT == 1 ? 4 : 3) : (D == 128 ? (NT == 1 ? 3 : 2) : 1);
    static constexpr int NS    = D == 64 ? (NT == 1 ? 3 : 4) : (D == 128 ? 2 : (NT == 1 ? 3 : 2));
    static constexpr int ND    = 4;                    // digits of q
    static constexpr int TILE  = KD_BLOCK * D;         // bytes of K or V
    static constexpr int HEAD  = 32;                   // scales and flags
    static constexpr int STAGE = 2 * TILE + HEAD;
    static constexpr int RING  = KD_WARPS * NS * STAGE;
    static constexpr int STATE = 2 * NT * 8 * 3 * 4;   // m, l, R
    static constexpr int FIXED = RING + STATE + NT * 8 * 4;
    // a segment's digits of q, [digit][row][dim], chunks swizzled like K's; at its end the merge buffer in their place.
    // (Beside them it left two CTAs an SM of three: F32, 48 sequences of up to 10240, D = 128, 8 rows a kv head 169 us
    // against 127; D = 64, 16 rows, F16, of up to 8000 tokens 84 against 69)
    static constexpr int Q     = ND * NT * 8 * D;
    static constexpr int OROW  = D + 4;                // floats per row of the merge buffer
    __host__ __device__ static constexpr int bytes(int rows) {
        return FIXED + (Q > 2 * rows * OROW * 4 ? Q : 2 * rows * OROW * 4);
    }
    static_assert(CTAS * (bytes(NT * 8) + KD_CTA_BYTES) <= KD_SM_BYTES, "the CTAs that the cuts count on do not fit on an SM");
    static_assert(FIXED % 16 == 0, "the digits are read by 16 bytes");
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

__device__ __forceinline__ void kd_mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// How units are cut: w = 0 flat, otherwise in parts of up to w blocks (one part where no unit is longer).
struct KdCut {
    int w;
    // items of a unit with nb blocks: blocks, or parts
    __device__ __forceinline__ int items(int nb) const { return w == 0 ? nb : (nb <= w ? 1 : (nb + w - 1) / w); }
};

// A walk over the segments (unit, blocks [b, e)) of a CTA's range of items.
struct KdWalk {
    int   s, u;  // sequence, unit of it
    int   b, e;
    int   left;  // items from this segment on
    KdSeq q;
    // to the next segment; false at the end of the range
    __device__ __forceinline__ bool next(const Kv8AttnParams & p, int units, KdCut cut) {
        left -= cut.w ? 1 : e - b;
        if (left <= 0) {
            return false;
        }
        b = 0;
        if (++u == units) {
            u = 0;
            s++;
            q = kd_seq(p, s);
        }
        e = cut.w ? q.nb : min(q.nb, left);  // parts of units run one per CTA: here units are whole
        return true;
    }
};

// A unit of which this CTA holds a part: its c0 .. c0 + n - 1 hold all of it.
struct KdPart {
    int s, u, c0, n;
};

// FS: each block's products summed from 0 (with PL); PL: the remainders of the weights too
template <int D, int NT, bool FS, bool PL, bool CAP>
__global__ void __launch_bounds__(KD_THREADS, KdSmem<D, NT>::CTAS) kv8_decode_kernel(const Kv8AttnParams p) {
    using L          = KdSmem<D, NT>;
    constexpr int NS = L::NS, ND = L::ND, CH = D / 64, MT = D / 16, E = D / 32, QR = NT * 8 / KD_WARPS;
    extern __shared__ __align__(16) char smem[];
    __shared__ int sh_last[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    char *    ring   = smem + warp * NS * L::STAGE;
    float *   state  = reinterpret_cast<float *>(smem + L::RING);     // [2][row][m, l, R]
    float *   qscale = state + 2 * NT * 8 * 3;                        // [row]
    char *    qf     = smem + L::FIXED;
    float *   obuf   = reinterpret_cast<float *>(smem + L::FIXED);    // [2][row][OROW], over the digits
    const int all_rows = p.ratio * p.n_q, groups = (all_rows + KD_ROWS - 1) / KD_ROWS;
    const int units = p.c.n_head_kv * groups;  // of a sequence
    kv8_dep_wait();

    // ---- this CTA's range: the sequences' items, scanned by every warp for itself
    KdWalk seg;
    KdCut  cut{ 0 };
    KdPart part[2];         // of the range's first and last segment
    int    total = 0, ctas = (int) gridDim.x, seq_first;  // seq_first: first item of sequence seg.s
    const int c = (int) blockIdx.x;
    {
        const int per = (p.t.n_seq + 31) / 32, s0 = min(lane * per, p.t.n_seq), s1 = min(s0 + per, p.t.n_seq);
        int       sum = 0, top = 0, one = 0;  // one: blocks of the lane's sequence, where it has only one
        for (int s = s0; s < s1; s++) {
            one = kd_seq(p, s).nb;
            sum += one, top = max(top, one);
        }
        total = (int) __reduce_add_sync(0xffffffffu, (unsigned) sum) * units;
        top   = (int) __reduce_max_sync(0xffffffffu, (unsigned) top);
        const int all = p.t.n_seq * units, spare = ctas - all;
        if (top <= KD_WHOLE) {
            cut.w = KD_WHOLE;
        } else if (spare > 0 && (int64_t) total * all <= (int64_t) KD_CROSS * ctas * spare) {
            cut.w = max(KD_PART, (total + spare - 1) / spare);
        } else if ((int64_t) ((all + ctas - 1) / ctas) * top * ctas <= total + (int64_t) KD_CROSS * ctas) {
            cut.w = top;
        }
        sum *= units;
        if (cut.w) {
            sum = per == 1 ? (s1 > s0 ? cut.items(one) * units : 0) : 0;
            for (int s = s0; s < s1 && per > 1; s++) {
                sum += cut.items(kd_seq(p, s).nb) * units;
            }
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, o);
            inc += lane >= o ? x : 0;
        }
        total = __shfl_sync(0xffffffffu, inc, 31);
        ctas  = min(ctas, total);
        if (c >= ctas) {
            return;
        }
        int each = 1, more = 0;
        if (ctas < total) {
            each = total / ctas, more = total - each * ctas;
        }
        const int begin = c * each + min(c, more);
        const int who   = __ffs(__ballot_sync(0xffffffffu, inc > begin)) - 1;  // its sequences hold the first item
        int       at    = __shfl_sync(0xffffffffu, inc - sum, who);
        int       s     = who * per;
        for (; per > 1; s += 32) {  // 32 of them at a time
            const int n  = s + lane < min((who + 1) * per, p.t.n_seq) ? cut.items(kd_seq(p, s + lane).nb) * units : 0;
            int       in = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, in, o);
                in += lane >= o ? x : 0;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at + in > begin);
            if (hit) {
                const int k = __ffs(hit) - 1;
                s += k;
                at = __shfl_sync(0xffffffffu, at + in - n, k);
                break;
            }
            at = __shfl_sync(0xffffffffu, at + in, 31);
        }
        seg.s = s;
        seg.q = kd_seq(p, s);
        seq_first = at;
        const int n = cut.items(seg.q.nb), off = begin - at;
        seg.u    = n == 1 ? off : off / n;
        seg.left = each + (c < more);
        const int k = off - seg.u * n;
        if (cut.w == 0) {
            seg.b = k;
            seg.e = min(seg.q.nb, k + seg.left);
        } else {  // parts that differ by one block at most
            const int base = n == 1 ? seg.q.nb : seg.q.nb / n, rest = seg.q.nb - base * n;
            seg.b = k * base + min(k, rest);
            seg.e = seg.b + base + (k < rest);
        }
        part[0] = KdPart{ 0, 0, 0, 0 }, part[1] = KdPart{ s, seg.u, c - k, cut.w ? n : 0 };
        if (n == 1) {
            part[1].n = 0;
        }
    }

    // ---- a segment's query rows rr = warp + 4 i, as they are: the first segment's before anything else
    uint32_t xr[QR][E];
    auto     load_q = [&] {
        const int h = seg.u / groups, r0 = (seg.u - h * groups) * KD_ROWS;
#pragma unroll
        for (int i = 0; i < QR; i++) {
            const int    r = r0 + warp + KD_WARPS * i, qi = (int) kv8_div((uint32_t) r, p.ratio_inv), hq = h * p.ratio + r - qi * p.ratio;
            const char * src = p.q.data + (int64_t) qi * p.q.nb1 + (int64_t) hq * p.q.nb2 + (int64_t) seg.s * p.q.nb3;
            const bool   live = r < all_rows && qi < seg.q.m;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int at = lane * E + e;
                xr[i][e]     = !live ? 0u : p.q.type == KV_F32 ? reinterpret_cast<const uint32_t *>(src)[at] : reinterpret_cast<const uint16_t *>(src)[at];
            }
        }
    };
    load_q();

    // ---- the warp's loads: block after block of the same walk, NS - 1 stages ahead.  Lane i holds the table entries
    // of the warp's i-th block from the cursor's base on, so that no load waits for a table entry but the first of 32
    KdWalk ld     = seg;
    int    ld_b   = ld.b + warp;
    bool   ld_on  = true;
    int    ld_i = 0, tab0 = -1, tab1 = -1;
    auto   fetch = [&] {
        const int k0 = (ld_b + KD_WARPS * lane) * KD_BLOCK, j = k0 >> p.c.log2p;
        const bool in = ld_b + KD_WARPS * lane < ld.e && k0 < ld.q.n;
        const int * row = p.t.pages + (int64_t) ld.s * p.t.stride;
        ld_i = 0;
        tab0 = in ? row[j] : -1;
        if (p.c.log2p == 4) {
            tab1 = in && k0 + 16 < ld.q.n ? row[j + 1] : -1;
        }
    };
    auto settle = [&] {  // brings the load cursor to a block of this warp, with its entries
        bool fresh = ld_i == 32;
        while (ld_on && ld_b >= ld.e) {
            ld_on = ld.next(p, units, cut);
            ld_b  = ld.b + warp;
            fresh = true;
        }
        if (ld_on && fresh) {
            fetch();
        }
    };
    // Places in a stage, less what a loop adds or flips (kd_swz of a row is what its lane gives, xor what the loop
    // gives): this lane's chunk of 512 bytes that are loaded; K's (and q's) chunk 2 t of row g; V's chunk g of row 2 t
    const uint32_t ld_to = (uint32_t) ((lane / (D / 16)) * D + (((lane % (D / 16)) ^ (D == 64 ? (lane >> 3) & 3 : lane / (D / 16))) << 4));
    const int      k_at  = g * D + (((D == 64 ? t : 2 * t) ^ kd_swz<D>(g)) << 4);
    const int      v_at  = 2 * t * D + (D == 64 ? (((g >> 1) ^ t) << 4) + (g & 1) * 8 : (g ^ (2 * t)) << 4);
    int  ld_stage = 0;
    auto load     = [&] {
        if (ld_on) {
            char *         st  = ring + ld_stage * L::STAGE;
            const int      h   = ld.u / groups;
            const int      row = (ld_b * KD_BLOCK) & (p.c.P - 1);  // of the block in its page
            int            pg0 = __shfl_sync(0xffffffffu, tab0, ld_i), pg1 = p.c.log2p == 4 ? __shfl_sync(0xffffffffu, tab1, ld_i) : pg0;
            const bool     ok0 = (unsigned) pg0 < (unsigned) p.c.n_pages, ok1 = (unsigned) pg1 < (unsigned) p.c.n_pages;
            pg0 = ok0 ? pg0 : 0, pg1 = ok1 ? pg1 : 0;
            const int64_t  ph0 = (int64_t) pg0 * p.c.n_head_kv + h, ph1 = (int64_t) pg1 * p.c.n_head_kv + h;
            const int64_t  o0 = (ph0 * p.c.P + row) * D;
            const int64_t  o1 = (p.c.log2p > 4 ? o0 : ph1 * p.c.P * D - 16 * D);
            const uint32_t z0 = ok0 ? 16u : 0u, z1 = ok1 ? 16u : 0u;
            const uint32_t dst = smem_addr(st);
            const int8_t * k0 = p.c.k + o0 + lane * 16, *k1 = p.c.k + o1 + lane * 16, *v0 = p.c.v + o0 + lane * 16, *v1 = p.c.v + o1 + lane * 16;
#pragma unroll
            for (int i = 0; i < 4 * CH; i++) {  // 32 rows of D / 16 chunks, 32 chunks at a time
                const bool     half = i >= 2 * CH;
                const uint32_t to   = dst + (ld_to ^ (uint32_t) ((D == 64 ? 0 : i * (512 / D) & 7) << 4)) + i * 512;
                kd_cp16(to, (half ? k1 : k0) + i * 512, half ? z1 : z0);
                kd_cp16(to + L::TILE, (half ? v1 : v0) + i * 512, half ? z1 : z0);
            }
            if (lane < 4) {
                const int64_t ph = lane & 1 ? ph1 : ph0;
                kd_cp4(dst + 2 * L::TILE + lane * 4, (lane < 2 ? p.c.k_scale : p.c.v_scale) + ph, (lane & 1 ? z1 : z0) / 4);
            } else if (lane < 6) {
                reinterpret_cast<int *>(st + 2 * L::TILE)[lane] = lane & 1 ? ok1 : ok0;
            }
            ld_b += KD_WARPS;
            ld_i++;
            settle();
        }
        ld_stage = ld_stage + 1 == NS ? 0 : ld_stage + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ld_i = 32;
    settle();
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
        load();
    }
    int           stage = 0;
    const int64_t slot  = (int64_t) KD_ROWS * (D + 4);  // floats of a part
    // dims lane * E .. + E of a result row: O (in units of 2^(R - KD_OFF)) over the sum (of 2^m); rows without
    // keys, and without a value scale, are 0
    auto emit = [&](int s, int h, int r, int nq, float (&v)[E], float mt, float lt, float rt) {
        const int qi = (int) kv8_div((uint32_t) r, p.ratio_inv), hq = h * p.ratio + r - qi * p.ratio;
        if (qi >= nq) {
            return;
        }
        const float inv = lt != 0.0f ? (1.0f / (1 << KD_OFF)) / lt : 0.0f, up = rt == -INFINITY ? 0.0f : kd_ex2(rt - mt);
#pragma unroll
        for (int e = 0; e < E; e++) {
            v[e] = v[e] * inv * up;
        }
        char * dst = p.o.data + (int64_t) hq * p.o.nb1 + (int64_t) qi * p.o.nb2 + (int64_t) s * p.o.nb3;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            if (p.o.type == KV_F32) {
                float * f = reinterpret_cast<float *>(dst) + lane * E + e;
                if (p.o.vec) {
                    *reinterpret_cast<float2 *>(f) = make_float2(v[e], v[e + 1]);
                } else {
                    f[0] = v[e], f[1] = v[e + 1];
                }
            } else {
                uint32_t w;
                if (p.o.type == KV_F16) {
                    w = kd_pack(v[e], v[e + 1]);
                } else {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[e], v[e + 1]);
                    w = *reinterpret_cast<const uint32_t *>(&b);
                }
                uint16_t * f = reinterpret_cast<uint16_t *>(dst) + lane * E + e;
                if (p.o.vec) {
                    *reinterpret_cast<uint32_t *>(f) = w;
                } else {
                    f[0] = (uint16_t) w, f[1] = (uint16_t) (w >> 16);
                }
            }
        }
    };

    for (bool more = true; more;) {
        const int  h = seg.u / groups, r0 = (seg.u - h * groups) * KD_ROWS;
        const int  rows  = min(all_rows - r0, min(KD_ROWS, NT * 8));
        const KdSeq sq   = seg.q;
        const int   low  = p.causal ? max(sq.n - (sq.m - 1), 0) : sq.n;  // keys below this are seen by every row
        // ---- the digits of q, row rr = warp + 4 i
        float xq[QR][E];
#pragma unroll
        for (int i = 0; i < QR; i++) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t u = xr[i][e];
                xq[i][e] = p.q.type == KV_F32 ? __uint_as_float(u) : p.q.type == KV_F16 ? __half2float(__ushort_as_half((uint16_t) u))
                                                                                       : __uint_as_float(u << 16);
            }
        }
#pragma unroll
        for (int i = 0; i < QR; i++) {
            const int rr   = warp + KD_WARPS * i;
            float     amax = 0.0f;
            bool      odd  = false;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float a = fabsf(xq[i][e]);
                amax          = fmaxf(amax, a);
                odd |= !(a < INFINITY);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            }
            odd = __any_sync(0xffffffffu, odd);
            // a power of two brings the largest element to [2^29, 2^30): the products are exact, and the fourth digit, with
            // what the others carry into it, stays below 128.  A row near the smallest numbers is brought up first, so that
            // the power is a number; one with an infinity or NaN gives NaN
            const float up  = amax < 0x1p-90f ? 0x1p64f : 1.0f;
            const int   ex  = min(max((int) (__float_as_uint(amax * up) >> 23) - 127, -90), 127);
            const float mul = __uint_as_float((uint32_t) (29 - ex + 127) << 23);
            if (lane == 0) {
                const float back = odd ? NAN : __uint_as_float((uint32_t) (ex - 29 + 127) << 23);
                qscale[rr]       = back * (CAP ? p.scale / p.softcap : p.scale * LOG2E) * (up == 1.0f ? 1.0f : 0x1p-64f);
            }
            uint32_t dig[ND][(E + 3) / 4];
#pragma unroll
            for (int d = 0; d < ND; d++) {
#pragma unroll
                for (int e = 0; e < (E + 3) / 4; e++) {
                    dig[d][e] = 0;
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                int v = odd ? 0 : __float2int_rn(xq[i][e] * up * mul);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const int low8 = (int8_t) v;  // digits in [-128, 127]
                    dig[d][e >> 2] |= (uint32_t) (low8 & 255) << (8 * (e & 3));
                    v = (v - low8) >> 8;
                }
            }
            const int at = rr * D + ((((lane * E) >> 4) ^ kd_swz<D>(rr)) << 4) + ((lane * E) & 15);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                char * to = qf + d * NT * 8 * D + at;
                if (E == 2) {
                    *reinterpret_cast<uint16_t *>(to) = (uint16_t) dig[d][0];
                } else {
#pragma unroll
                    for (int e = 0; e < E / 4; e++) {
                        reinterpret_cast<uint32_t *>(to)[e] = dig[d][e];
                    }
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
                const int rr = nt * 8 + 2 * t + i, qi = (int) kv8_div((uint32_t) (r0 + rr), p.ratio_inv);
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
            // S^T = K Q^T: keys 16a + g and 16a + g + 8 of lane g, in the chunks of lane t
            // (one half of the keys at a time where two columns of rows would need more registers than there are)
            constexpr int AP = NT == 1 ? 2 : 1;
#pragma unroll
            for (int a0 = 0; a0 < 2; a0 += AP) {
                int acc[AP][NT][ND][4];
#pragma unroll
                for (int i = 0; i < AP * NT * ND * 4; i++) {
                    (&acc[0][0][0][0])[i] = 0;
                }
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    const int at = (k_at ^ ((j & 1) << 4)) + (j >> 1) * 128;
                    uint4     w[AP][2];
#pragma unroll
                    for (int a = 0; a < AP; a++) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            w[a][i] = *reinterpret_cast<const uint4 *>(st + (16 * (a0 + a) + 8 * i) * D + at);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int d = 0; d < ND; d++) {
                            const uint4 b = *reinterpret_cast<const uint4 *>(qf + (d * NT + nt) * 8 * D + at);
#pragma unroll
                            for (int a = 0; a < AP; a++) {
                                kd_mma_s8(acc[a][nt][d], w[a][0].x, w[a][1].x, w[a][0].y, w[a][1].y, b.x, b.y);
                                kd_mma_s8(acc[a][nt][d], w[a][0].z, w[a][1].z, w[a][0].w, w[a][1].w, b.z, b.w);
                            }
                        }
                    }
                }
#pragma unroll
                for (int a = 0; a < AP; a++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            // |digit dots| < 2^22 (D = 256): two of them fit an int
                            const float lo   = (float) (acc[a][nt][1][e] * 256 + acc[a][nt][0][e]);
                            s[a0 + a][nt][e] = fmaf((float) (acc[a][nt][3][e] * 256 + acc[a][nt][2][e]), 65536.0f, lo);
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
                        if (CAP) {
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
                        if (PL) {
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
            // (FS: both halves of the keys side by side, where registers allow)
            const char * vt = st + L::TILE;
            constexpr int WORDS = D == 64 ? 2 : 4, AV = FS && (D <= 128 || NT == 1) ? 2 : 1;
#pragma unroll
            for (int a0 = 0; a0 < 2; a0 += AV) {
#pragma unroll
                for (int j = 0; j < (D + 127) / 128; j++) {
                    uint32_t w[AV][4][WORDS];
#pragma unroll
                    for (int a = 0; a < AV; a++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r = (16 * (a0 + a) + (i & 1) + 8 * (i >> 1)) * D;  // beyond row 2 t
                            if (D == 64) {
                                const uint2 u = *reinterpret_cast<const uint2 *>(vt + r + v_at);
                                w[a][i][0] = u.x, w[a][i][1] = u.y;
                            } else {
                                const uint4 u = *reinterpret_cast<const uint4 *>(vt + r + (v_at ^ ((i & 1) << 4)) + 128 * j);
                                w[a][i][0] = u.x, w[a][i][1] = u.y, w[a][i][WORDS - 2] = u.z, w[a][i][WORDS - 1] = u.w;
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < WORDS; k++) {
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            float x[NT][4];
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
                            }
#pragma unroll
                            for (int a = 0; a < AV; a++) {
                                const uint32_t x0 = w[a][0][k] ^ 0x80808080u, x1 = w[a][1][k] ^ 0x80808080u;
                                const uint32_t x2 = w[a][2][k] ^ 0x80808080u, x3 = w[a][3][k] ^ 0x80808080u;
                                const uint32_t y = kd_prmt(x0, x1, q ? 0x7362 : 0x5140), z = kd_prmt(x2, x3, q ? 0x7362 : 0x5140);
                                const uint32_t f[4] = { kd_half2(y, 0x4140), kd_half2(y, 0x4342), kd_half2(z, 0x4140), kd_half2(z, 0x4342) };
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    float(&to)[4] = FS ? x[nt] : o[j * 8 + 2 * k + q][nt];
                                    if (PL) {
                                        kd_mma(to, f, pl[a0 + a][nt][0], pl[a0 + a][nt][1]);
                                    }
                                    kd_mma(to, f, ph[a0 + a][nt][0], ph[a0 + a][nt][1]);
                                }
                            }
                            if (FS) {
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    float(&to)[4] = o[j * 8 + 2 * k + q][nt];
                                    f2unpack(fadd2(f2pack(to[0], to[1]), f2pack(x[nt][0], x[nt][1])), to[0], to[1]);
                                    f2unpack(fadd2(f2pack(to[2], to[3]), f2pack(x[nt][2], x[nt][3])), to[2], to[3]);
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
#pragma unroll 1
        for (int round = 0; round < 2; round++) {
            __syncthreads();  // the digits are not read any more; then: the two states are there
            if ((warp < 2) == (round == 1)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int rr = nt * 8 + 2 * t + i;
                        float *   st = state + ((warp & 1) * NT * 8 + rr) * 3;
                        float *   w  = obuf + ((warp & 1) * rows + rr) * L::OROW + (D == 64 ? 8 : 16) * g;
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
                                float4 v = make_float4(o[2 * j][nt][i], o[2 * j][nt][i + 2], o[2 * j + 1][nt][i], o[2 * j + 1][nt][i + 2]);
                                float4 * to = reinterpret_cast<float4 *>(w + (j >> 2) * 128 + 4 * (j & 3));
                                if (round == 1) {
                                    const float4 y = *to;
                                    v.x = v.x * fa + y.x * fb, v.y = v.y * fa + y.y * fb;
                                    v.z = v.z * fa + y.z * fb, v.w = v.w * fa + y.w * fb;
                                }
                                *to = v;
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = seg.b == 0 && seg.e == sq.nb;
        // two states left: to dst, or, of a part of a unit, to the workspace
#pragma unroll 1
        for (int rr = warp; rr < rows; rr += KD_WARPS) {
            const float * za = state + rr * 3, *zb = za + NT * 8 * 3;
            const float * ya = obuf + rr * L::OROW + lane * E, *yb = ya + rows * L::OROW;
            const float   mt = fmaxf(za[0], zb[0]), rt = fmaxf(za[2], zb[2]);
            const float   ms = mt == -INFINITY ? 0.0f : mt, rs = rt == -INFINITY ? 0.0f : rt;
            const float   lt = za[1] * kd_ex2(za[0] - ms) + zb[1] * kd_ex2(zb[0] - ms), fa = kd_ex2(za[2] - rs), fb = kd_ex2(zb[2] - rs);
            float         v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = ya[e] * fa + yb[e] * fb;
            }
            if (whole) {
                emit(seg.s, h, r0 + rr, sq.m, v, mt, lt, rt);
            } else {
                float * w = p.part + (2 * c + (seg.b == 0)) * slot + rr * (D + 4);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    w[lane * E + e] = v[e];
                }
                if (lane == 0) {
                    *reinterpret_cast<float4 *>(w + D) = make_float4(mt, lt, rt, 0.0f);
                }
            }
        }
        if (!whole && cut.w == 0) {
            // the CTAs that hold a part: the first `over` ranges are one block longer than `each`
            const int  each = total / ctas, over = total - each * ctas, first = seq_first + seg.u * sq.nb;
            const auto cta_of = [&](int x) { return x < over * (each + 1) ? x / (each + 1) : over + (x - over * (each + 1)) / each; };
            const int  c0 = cta_of(first);
            part[0] = part[1], part[1] = KdPart{ seg.s, seg.u, c0, cta_of(first + sq.nb - 1) - c0 + 1 };
        }
        const int s_before = seg.s;
        more               = seg.next(p, units, cut);
        if (more && seg.s != s_before) {
            seq_first += sq.nb * units;  // of use in a flat cut only
        }
        if (more) {
            load_q();
        }
        __syncthreads();  // state, obuf and the Q digits are written again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (part[0].n + part[1].n == 0) {
        return;
    }

    // ---- the parts of a unit, joined by the last CTA that arrives
    __threadfence();
    __syncthreads();
    if (tid < 2) {
        const KdPart & x = tid ? part[1] : part[0];
        sh_last[tid]     = x.n && atomicAdd(&p.counters[x.c0], 1u) == (uint32_t) (x.n - 1);
        if (sh_last[tid]) {
            p.counters[x.c0] = 0;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        if (!sh_last[i]) {
            continue;
        }
        __threadfence();
        const KdPart x  = i ? part[1] : part[0];
        const int    h = x.u / groups, r0 = (x.u - h * groups) * KD_ROWS, rows = min(all_rows - r0, min(KD_ROWS, NT * 8));
        const int    nq = kd_seq(p, x.s).m;
#pragma unroll 1
        for (int rr = warp; rr < rows; rr += KD_WARPS) {
            const float * w  = p.part + 2 * x.c0 * slot + rr * (D + 4);
            float         mt = -INFINITY, rt = -INFINITY, lt = 0.0f, v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = 0.0f;
            }
#pragma unroll 1
            for (int k0 = 0; k0 < x.n; k0 += 32) {
                // a part's state per lane: its factor, and the row's sum
                const int  k = k0 + lane;
                float4     z = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                if (k < x.n) {
                    z = __ldcg(reinterpret_cast<const float4 *>(w + (2 * k + (k == 0)) * slot + D));
                }
                float mn = z.x, rn = z.z;
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
                    rn = fmaxf(rn, __shfl_xor_sync(0xffffffffu, rn, o));
                }
                mn = fmaxf(mn, mt), rn = fmaxf(rn, rt);
                const float ms = mn == -INFINITY ? 0.0f : mn, rs = rn == -INFINITY ? 0.0f : rn;
                const float f = kd_ex2(z.z - rs), f0 = kd_ex2(rt - rs);
                float       ls = z.y * kd_ex2(z.x - ms);
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    ls += __shfl_xor_sync(0xffffffffu, ls, o);
                }
                lt = lt * kd_ex2(mt - ms) + ls;
                mt = mn, rt = rn;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    v[e] *= f0;
                }
                constexpr int B = E == 8 ? 8 : 16;  // parts in flight
                const int     n = min(x.n - k0, 32);
#pragma unroll 1
                for (int j = 0; j < n; j += B) {
                    float y[B][E];
#pragma unroll
                    for (int b = 0; b < B; b++) {
                        const int     kk = k0 + j + b;
                        const float * src = w + (2 * kk + (kk == 0)) * slot + lane * E;
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float2 u = j + b < n ? __ldcg(reinterpret_cast<const float2 *>(src + e)) : make_float2(0.0f, 0.0f);
                            y[b][e] = u.x, y[b][e + 1] = u.y;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < B; b++) {
                        const float fb = __shfl_sync(0xffffffffu, f, (j + b) & 31);
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            v[e] += y[b][e] * fb;
                        }
                    }
                }
            }
            emit(x.s, h, r0 + rr, nq, v, mt, lt, rt);
        }
    }
}

namespace {

template <int D, int NT, bool FS, bool PL, bool CAP>
cudaError_t launch_one(const Kv8AttnParams & p, unsigned ctas, int rows, cudaStream_t stream) {
    const size_t smem = KdSmem<D, NT>::bytes(rows);
    static Kv8Once once;
    const cudaError_t e = once.smem(kv8_decode_kernel<D, NT, FS, PL, CAP>, KdSmem<D, NT>::bytes(NT * 8));
    return e != cudaSuccess ? e : kv8_launch(kv8_decode_kernel<D, NT, FS, PL, CAP>, dim3(ctas), KD_THREADS, smem, stream, p);
}

template <int D, int NT, bool CAP>
cudaError_t launch_nt(const Kv8AttnParams & p, unsigned ctas, int rows, cudaStream_t stream) {
    const bool fresh = p.o.type == KV_F32 || (int64_t) p.t.max_pages * p.c.P > KD_LONG;
    return fresh                ? launch_one<D, NT, true, true, CAP>(p, ctas, rows, stream)
           : p.o.type == KV_F16 ? launch_one<D, NT, false, true, CAP>(p, ctas, rows, stream)
                                : launch_one<D, NT, false, false, CAP>(p, ctas, rows, stream);
}

template <int D>
cudaError_t launch_d(const Kv8AttnParams & p, unsigned ctas, int rows, cudaStream_t stream) {
    if (p.softcap > 0.0f) {
        return rows <= 8 ? launch_nt<D, 1, true>(p, ctas, rows, stream) : launch_nt<D, 2, true>(p, ctas, rows, stream);
    }
    return rows <= 8 ? launch_nt<D, 1, false>(p, ctas, rows, stream) : launch_nt<D, 2, false>(p, ctas, rows, stream);
}

// CTAs that an SM holds at once: what KdSmem plans for
constexpr int KD_CTAS_MOST = KdSmem<64, 1>::CTAS;

// (with the status within the 64 KiB that a caller has zeroed)
size_t counter_bytes(int sms) {
    return ((size_t) sms * KD_CTAS_MOST * 4 + 255) / 256 * 256;
}

int ctas_per_sm(int D, int rows) {
    return rows <= 8 ? (D == 64 ? KdSmem<64, 1>::CTAS : D == 128 ? KdSmem<128, 1>::CTAS : KdSmem<256, 1>::CTAS)
                     : (D == 64 ? KdSmem<64, 2>::CTAS : D == 128 ? KdSmem<128, 2>::CTAS : KdSmem<256, 2>::CTAS);
}

// The kernel for many rows (D <= 128) takes a call that gives every SM of each wave of its CTAs five units of this
// kernel for two, a part of a block's keys counted like the whole.  BF16, D = 128, this kernel against that at 1.7 such
// units per SM (4 sequences of 4096, 32 rows per kv head): 39 us against 35; at 2.0 (one of 8192, 32 rows) 30 against 36; at
// 2.6 (16 of 1024, 48 rows) 52 against 31; at 3.5 (4 of 4096, 64 rows) 65 against 35; at 3.9 (one of 8192, 64 rows) 38
// against 36, and of 256 rows 99 against 46.  F32: 54 against 37 at 2.6, 69 against 41 at 3.5, 40 against 38 at 3.9; F16 with
// D = 64: 31 against 25 at 2.6.  The host knows the table's capacity, not the lengths: two sequences of 100 tokens in
// tables for 8192 (48 rows, F32) count 9 parts each and take 14 us here against 10.
bool many_rows(Kv8AttnParams & p, int sms) {
    const int64_t heads = (int64_t) p.t.n_seq * p.c.n_head_kv, rows = (int64_t) p.ratio * p.n_q;
    const int     tile  = kv8_dense_tile(p);
    const int64_t items = heads * ((rows + tile - 1) / tile), waves = (items + sms - 1) / sms;
    p.parts             = kv8_dense_parts(items, (int64_t) p.t.max_pages * p.c.P, sms);
    return p.c.D <= 128 && heads * ((rows + KD_ROWS - 1) / KD_ROWS) * p.parts * 2 >= 5 * waves * sms;
}

}  // namespace

// Counters (one per CTA, in a place of one size for every shape: a workspace serves them all, and no shape's
// partial results may lie on another's counters) and two partial results per CTA, whatever the lengths are, or
// those of the kernel for many rows.
size_t kv8_attn_workspace_bytes(int D, int64_t rows, int64_t heads, int64_t tokens, int sms) {
    size_t most = 2 * (size_t) sms * (size_t) ctas_per_sm(D, (int) rows) * KD_ROWS * (size_t) (D + 4) * 4;
    for (int tile = 128; tile <= 256 && D <= 128; tile += 128) {
        const int64_t items = heads * ((rows + tile - 1) / tile);
        most                = std::max(most, kv8_dense_part_bytes(D, items, tile, kv8_dense_parts(items, tokens, sms)));
    }
    return WS_STATUS_BYTES + counter_bytes(sms) + most;
}

cudaError_t launch_kv8_attn(const Kv8AttnParams & p0, int sms, cudaStream_t stream) {
    Kv8AttnParams p    = p0;
    p.ratio_inv        = p.ratio == 1 ? 0u : (uint32_t) ((1ull << 32) / (uint64_t) p.ratio + 1);
    p.counters = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(p.status) + WS_STATUS_BYTES);
    p.part     = reinterpret_cast<float *>(reinterpret_cast<char *>(p.counters) + counter_bytes(sms));
    if (many_rows(p, sms)) {
        return launch_kv8_dense(p, stream);
    }
    const int     most = sms * ctas_per_sm(p.c.D, p.ratio * p.n_q);
    const int     all = p.ratio * p.n_q, rows = all < KD_ROWS ? all : KD_ROWS;
    const int64_t units  = (int64_t) p.t.n_seq * p.c.n_head_kv * ((all + KD_ROWS - 1) / KD_ROWS);
    const int64_t blocks = units * (((int64_t) p.t.max_pages * p.c.P + KD_BLOCK - 1) / KD_BLOCK);  // at most
    if (blocks > INT32_MAX) {
        return cudaErrorInvalidValue;  // refused by the caller's checks
    }
    const unsigned ctas  = (unsigned) (blocks < most ? blocks : most);
    switch (p.c.D) {
        case 64:
            return launch_d<64>(p, ctas, rows, stream);
        case 128:
            return launch_d<128>(p, ctas, rows, stream);
        default:
            return launch_d<256>(p, ctas, rows, stream);
    }
}

}  // namespace mm3fa
