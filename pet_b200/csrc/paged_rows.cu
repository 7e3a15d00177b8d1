// Attention of a few query rows over a paged cache: single tokens, draft tokens, and every call in fp32.
//
//   out[row] = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),   t_j = scale log2(e) q[row] . k_j,   m = max_j t_j
//
// A tile is 16 rows = (token, query head) pairs that share one key head, so a key is read once for all the heads it serves.  A CTA
// is four warps; a step of it is 4 x CK keys, CK of them (16 halves, 8 floats) per warp, and every warp runs by itself: its
// own ring of stages filled by its own 16-byte asynchronous copies, its own running maximum, sum and 16 x DP accumulators in
// registers.  The warps meet once, at the end of a tile.  Bound by HBM: per 16 keys of width 128 a warp issues 32
// mma.sync.m16n8k16 and 16 ldmatrix beside 8 KB of loads; 48 % of the issue slots are used over a whole call.  (A 16-row tile
// would leave seven eighths of a 128-row tcgen05 tile empty; paged_tiles.cu takes over where there are rows for it.)
//
// Work is split by ranges: the key steps of all (sequence, row tile, key head) units are laid end to end and every CTA takes an
// equal share, whatever the lengths; a unit that crosses a border leaves one piece per CTA, and k_paged_join adds the pieces in order.
// Few units of moderate length go to a thread-block cluster each instead, which adds its sums through shared memory; many units, or
// units of a few steps, to a CTA each.  64 sequences of up to 8000 keys (1.05 GB): 182 to 188 us,
// 5.6 to 5.8 TB/s; one token on 1500 keys: 11 us a call.
//
// fp32 runs on the TF32 tensor cores (up to four rows: on multiply-adds, see FewRows) with both operands split in two (x = hi + lo, hi the
// upper 11 bits: hi hi + hi lo + lo hi, 2^-21 of a product left out), and the product with V starts from zero for every 8 keys and is added
// in registers, since a tensor core's own accumulation cuts off instead of rounding.  Scores, statistics and sums are fp32 for every type;
// probabilities are rounded to the cache's type for the second product (16-bit types; the sum of the row takes them unrounded).  Prompts
// in fp32 fetch and split their keys again for every 16 rows: 2000 tokens x 12 heads of 64 take 343 us and 11 of joining, the tensor pipe
// 25 % busy and 41 % of the issue slots used (629 instructions of a warp per 8 keys, 48 of them products).
//
// Rows that see no key give zeros.  A masked key never contributes, whatever its value: its score is replaced before the
// maximum, and non-finite values of its v are taken out of the stage before the product (see `scrub`).  Infinities that are seen give what
// the formula gives: a score of -inf weighs nothing, one of +inf makes the row NaN, an infinite v is its column's result.
#include "paged.cuh"
#include "tc_ptx.cuh"
#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace petb200 {
namespace {

constexpr int kRowWarps = 4, kRowThreads = 32 * kRowWarps, kRows = 16;

template <typename T, int DP> struct RowCfg {
    static constexpr bool f32 = sizeof(T) == 4;
    static constexpr int CK = f32 ? 8 : 16;                 // keys of a warp's step
    static constexpr int KT = CK * kRowWarps;               // keys of a CTA's step
    static constexpr int CPR = DP * (int)sizeof(T) / 16;    // 16-byte pieces of a row
    static constexpr int RPI = 32 / CPR;                    // rows that one copy instruction of the warp covers
    static constexpr int NI = CK / RPI;                     // copy instructions per operand and step
    static constexpr int HALF = CK * DP * (int)sizeof(T);   // bytes of one operand's stage
    // Blocks per SM, and stages of a warp's ring: three blocks of two stages at 168 registers a thread, or two of three at 255, take the
    // same time over long sequences (184 us for 64 of up to 8000 keys); short ones gain from the third block (128 of up to 500 keys behind
    // a prefix: 117 -> 114 us).  fp32's hi and lo queries of 128 values spill at 168.
    static constexpr int CTAS = DP == 128 && f32 ? 2 : 3, NST = DP == 64 ? 4 : f32 ? 3 : 2;
    static constexpr int MP = DP + 8;                       // pitch of a row of sums where the warps meet: eight rows, eight banks
    static constexpr int WARP_BYTES = 2 * HALF * NST;
    static constexpr int SMEM = WARP_BYTES * kRowWarps;
    static_assert(WARP_BYTES >= kRows * (MP + 2) * 4, "a warp's stages hold its accumulators when the warps meet");
    static_assert(SMEM * CTAS <= 224 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo with hi the upper 11 bits of x.  lo is NaN where x is not finite, so that a step with such a value shows in its sums.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t &hi, uint32_t &lo) {
    hi = x & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// The two parts where x may be infinite: `hi` has it in the product of the upper parts, `cross` (0 there) goes with the other operand's lo, which
// may be 0.
__device__ __forceinline__ void split_careful(uint32_t x, uint32_t &hi, uint32_t &lo, uint32_t &cross) {
    split_tf32(x, hi, lo);
    const bool inf = (x & 0x7fffffffu) == 0x7f800000u;
    lo = inf ? 0u : lo, cross = inf ? 0u : hi;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value)
        return ptx::pack_f16x2(a, b);
    else
        return ptx::pack_bf16x2(a, b);
}
template <typename T> __device__ __forceinline__ bool finite(T v) {
    const float f = to_f32(v);
    return fabsf(f) <= FLT_MAX;
}

// a + b, at most 2^32 - 1: starts that run backwards may claim any amount of work, and a sum that wrapped round would place it wrongly.
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return a + min(b, ~a); }
// Sum of `x` over the threads before this one, and over all of them in `total`.
__device__ __forceinline__ unsigned block_scan(unsigned x, unsigned &total, unsigned *tmp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
        inc = add_sat(inc, lane >= o ? v : 0u);
    }
    __syncthreads(); // (tmp of an earlier scan has been read)
    if (lane == 31)
        tmp[warp] = inc;
    const unsigned up = __shfl_up_sync(0xffffffffu, inc, 1);
    __syncthreads();
    unsigned before = lane ? up : 0u;
    total = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        before = add_sat(before, w < warp ? tmp[w] : 0u);
        total = add_sat(total, tmp[w]);
    }
    return before;
}

enum { kModeRanges = 0, kModeUnits = 1, kModePieces = 2, kModeCluster = 3 };

// One unit: rows [16 rt, 16 rt + 16) of sequence b's (token, head) pairs on key head h.
struct Unit {
    int b, rt, h, t0, ql, own, n; // n: keys that its last row sees
    int skip;                     // shared keys that come before them elsewhere
};

template <typename T, int DP> struct RowTile {
    using C = RowCfg<T, DP>;
    static constexpr int NJ = C::CK / 8;
    static constexpr int QR = C::f32 ? DP / 8 * 8 : DP / 16 * 4; // registers of the query fragments (fp32: hi and lo)

    float o[DP / 8][4];
    float m[2], l[2];

    __device__ __forceinline__ static int swz(int row, int piece) { return piece ^ (row & 7); }

    // Issues the copies of keys [base, base + CK) of the unit; keys from `n` on are zeros.
    __device__ __forceinline__ static void fetch(const PagedArgs &a, const Unit &u, uint32_t stage, int base, int n) {
        const int lane = threadIdx.x & 31;
        long long ko = -1, vo = 0;
        if (lane < C::CK && base + lane < n) {
            int slot;
            const int p = a.s.page(u.b, base + lane + u.skip, slot);
            if (p >= 0) {
                ko = (long long)p * a.kp + (long long)slot * a.ks + (long long)u.h * a.kh;
                vo = (long long)p * a.vp + (long long)slot * a.vs + (long long)u.h * a.vh;
            }
        }
        const int piece = lane % C::CPR;
        const T *kc = (const T *)a.kc, *vc = (const T *)a.vc;
        const bool col = piece * (16 / (int)sizeof(T)) < a.dim;
#pragma unroll
        for (int i = 0; i < C::NI; ++i) {
            const int row = i * C::RPI + lane / C::CPR;
            const long long k = __shfl_sync(0xffffffffu, ko, row), v = __shfl_sync(0xffffffffu, vo, row);
            const int bytes = col && k >= 0 ? 16 : 0;
            const long long at = piece * (16 / (int)sizeof(T));
            const uint32_t dst = stage + row * (DP * (int)sizeof(T)) + swz(row, piece) * 16;
            cp_async_16_or_zero(dst, bytes ? kc + k + at : kc, bytes);
            cp_async_16_or_zero(dst + C::HALF, bytes ? vc + v + at : vc, bytes);
        }
    }

    // Query fragments of the tile, straight from the rows.
    __device__ __forceinline__ static void load_q(const PagedArgs &a, const Unit &u, uint32_t (&qf)[QR]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const T *p[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = u.rt * kRows + g + 8 * r, tok = row / a.group, hd = row - tok * a.group;
            p[r] = tok < u.ql ? (const T *)a.q + (long long)(u.t0 + tok) * a.q_tok + (long long)(u.h * a.group + hd) * a.q_head : nullptr;
        }
        if constexpr (C::f32) {
#pragma unroll
            for (int k = 0; k < DP / 8; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) { // a0 (g, c) a1 (g + 8, c) a2 (g, c + 4) a3 (g + 8, c + 4)
                    const int d = k * 8 + c + (e >> 1) * 4;
                    const float x = p[e & 1] && d < a.dim ? __ldg((const float *)p[e & 1] + d) : 0.f;
                    split_tf32(__float_as_uint(x), qf[k * 8 + e], qf[k * 8 + 4 + e]);
                }
        } else {
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = k * 16 + 2 * c + (e >> 1) * 8;
                    qf[k * 4 + e] = p[e & 1] && d < a.dim ? __ldg((const unsigned *)(p[e & 1] + d)) : 0u;
                }
        }
    }

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int t = 0; t < DP / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[t][e] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // Column of accumulator o[t][e] (fp32 spreads a lane's columns so that v is read 16 bytes at a time).
    __device__ __forceinline__ static int column(int t, int e) {
        const int c = threadIdx.x & 3;
        return C::f32 ? (t >> 2) * 32 + 8 * c + 4 * (e & 1) + (t & 3) : t * 8 + 2 * c + (e & 1);
    }

    // Non-finite values of v in a step whose keys some rows do not see (a product with probability 0 would be NaN), in fp32 in any step (so
    // would one with a lower part of 0).  They are added where they are seen (an infinity or a NaN outlives any factor) and taken out of
    // the stage.
    __device__ __forceinline__ void scrub(unsigned char *vst, int base, int lim0, int lim1) {
        const int lane = threadIdx.x & 31;
        T *v = reinterpret_cast<T *>(vst);
        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll 1
        for (int r = 0; r < C::CK; ++r)
#pragma unroll
            for (int t = 0; t < DP / 8; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = column(t, e);
                    const T x = v[(r * C::CPR + swz(r, d / E)) * E + d % E];
                    if (!finite(x)) {
                        o[t][e] += base + r < lim0 ? to_f32(x) : 0.f;
                        o[t][e + 2] += base + r < lim1 ? to_f32(x) : 0.f;
                    }
                }
        __syncwarp();
        for (int i = lane; i < C::CK * DP; i += 32)
            if (!finite(v[i]))
                v[i] = from_f32<T>(0.f);
        __syncwarp();
    }

    // fp32: the scores of the stage's eight keys.  CAREFUL: right for infinite keys too.  (A query with an infinity is NaN either way: all its
    // scores are infinite or NaN.)
    template <bool CAREFUL> __device__ __forceinline__ static void scores_f32(const uint32_t (&qf)[QR], uint32_t stage, float (&s)[4]) {
        const int lane = threadIdx.x & 31, row = lane & 7;
        float x[3][4];
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[i][e] = 0.f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) { // two k steps of 8 per ldmatrix: pieces 4 k .. 4 k + 3 of the 8 keys
            uint32_t r[4];
            ldsm4(stage + row * (DP * 4) + swz(row, 4 * k + (lane >> 3)) * 16, r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t bh[2], bl[2], bx[2], qh[4], ql[4];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (CAREFUL)
                        split_careful(r[2 * h + e], bh[e], bl[e], bx[e]);
                    else
                        split_tf32(r[2 * h + e], bh[e], bl[e]), bx[e] = bh[e];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    qh[e] = qf[(2 * k + h) * 8 + e], ql[e] = qf[(2 * k + h) * 8 + 4 + e];
                mma8(x[0], qh, bh[0], bh[1]);
                mma8(x[1], qh, bl[0], bl[1]);
                mma8(x[2], ql, bx[0], bx[1]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s[e] = x[0][e] + (x[1][e] + x[2][e]);
    }

    // One step: keys [base, base + CK) in `stage`; row g sees keys below lim0, row g + 8 below lim1.
    __device__ __forceinline__ void step(const PagedArgs &a, const uint32_t (&qf)[QR], uint32_t stage, unsigned char *stage_p, int base,
                                         int lim0, int lim1, bool masked) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        float s[NJ][4];
        if constexpr (C::f32) {
            scores_f32<false>(qf, stage, s[0]);
            // A value that is not finite makes its sums NaN through its lower part: such a step is done again with infinities kept out of the
            // cross products, since 0 x infinity is not what the formula has there.
            if (__any_sync(0xffffffffu, s[0][0] != s[0][0] || s[0][1] != s[0][1] || s[0][2] != s[0][2] || s[0][3] != s[0][3]))
                scores_f32<true>(qf, stage, s[0]);
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[j][e] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t r[4]; // (keys 0-7, k 0-7) (0-7, 8-15) (8-15, 0-7) (8-15, 8-15)
                const int row = (lane & 7) + ((lane >> 4) << 3);
                ldsm4(stage + row * (DP * 2) + swz(row, 2 * k + ((lane >> 3) & 1)) * 16, r);
                uint32_t qq[4] = {qf[4 * k], qf[4 * k + 1], qf[4 * k + 2], qf[4 * k + 3]};
                mma16<T>(s[0], qq, r[0], r[1]);
                mma16<T>(s[1], qq, r[2], r[3]);
            }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[j][e] *= a.sl2, s[j][e + 2] *= a.sl2;
                if (masked) {
                    const int key = base + j * 8 + 2 * c + e;
                    s[j][e] = key < lim0 ? s[j][e] : -INFINITY;
                    s[j][e + 2] = key < lim1 ? s[j][e + 2] : -INFINITY;
                }
                mx0 = fmaxf(mx0, s[j][e]), mx1 = fmaxf(mx1, s[j][e + 2]);
            }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
        }
        mx0 = lifted<T>(mx0, 15.f), mx1 = lifted<T>(mx1, 15.f);
        if (__any_sync(0xffffffffu, mx0 > m[0] || mx1 > m[1])) {
            const float n0 = fmaxf(m[0], mx0), n1 = fmaxf(m[1], mx1);
            const float f0 = m[0] == n0 ? 1.f : exp2_approx(m[0] - n0), f1 = m[1] == n1 ? 1.f : exp2_approx(m[1] - n1);
            m[0] = n0, m[1] = n1;
            l[0] *= f0, l[1] *= f1;
#pragma unroll
            for (int t = 0; t < DP / 8; ++t)
                o[t][0] *= f0, o[t][1] *= f0, o[t][2] *= f1, o[t][3] *= f1;
        }
        const float z0 = m[0] == -INFINITY ? 0.f : m[0], z1 = m[1] == -INFINITY ? 0.f : m[1]; // (nothing seen so far: every power is 0)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[j][e] = exp2_approx(s[j][e] - z0), s[j][e + 2] = exp2_approx(s[j][e + 2] - z1);
                l[0] += s[j][e], l[1] += s[j][e + 2];
            }
        if (!C::f32 && masked) {
            bool bad = false;
            const uint4 *v = reinterpret_cast<const uint4 *>(stage_p + C::HALF);
            for (int i = lane; i < C::CK * C::CPR; i += 32) {
                const uint4 w = v[i];
                const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(T); ++e)
                    bad |= !finite(x[e]);
            }
            if (__any_sync(0xffffffffu, bad))
                scrub(stage_p + C::HALF, base, lim0, lim1);
        }
        if constexpr (C::f32) {
            // k index c of the product is key 2 c, c + 4 is key 2 c + 1: the scores are where the product wants them
            uint32_t ph[4], pl[4];
            split_tf32(__float_as_uint(s[0][0]), ph[0], pl[0]);
            split_tf32(__float_as_uint(s[0][2]), ph[1], pl[1]);
            split_tf32(__float_as_uint(s[0][1]), ph[2], pl[2]);
            split_tf32(__float_as_uint(s[0][3]), ph[3], pl[3]);
            const unsigned char *vst = stage_p + C::HALF;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) { // lane g's column of tile 4 i + e is 32 i + 4 g + e
                const int r0 = 2 * c, r1 = 2 * c + 1;
                uint32_t h0[4], l0[4], h1[4], l1[4];
                auto load = [&]() { // answers whether all of it is finite
                    const uint4 w0 = *reinterpret_cast<const uint4 *>(vst + r0 * (DP * 4) + swz(r0, 8 * i + g) * 16);
                    const uint4 w1 = *reinterpret_cast<const uint4 *>(vst + r1 * (DP * 4) + swz(r1, 8 * i + g) * 16);
                    const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        split_tf32(x0[e], h0[e], l0[e]);
                        split_tf32(x1[e], h1[e], l1[e]);
                        sum += __uint_as_float(l0[e]) + __uint_as_float(l1[e]);
                    }
                    return sum == sum;
                };
                if (__any_sync(0xffffffffu, !load())) { // (none of the columns before had such a value, and none behind has one any more)
                    scrub(stage_p + C::HALF, base, lim0, lim1);
                    load();
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y[4] = {0.f, 0.f, 0.f, 0.f};
                    mma8(y, pl, h0[e], h1[e]);
                    mma8(y, ph, l0[e], l1[e]);
                    mma8(y, ph, h0[e], h1[e]);
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        o[4 * i + e][z] += y[z];
                }
            }
        } else {
            const uint32_t p[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                uint32_t r[4]; // (keys 0-7, cols 0-7) (keys 8-15, cols 0-7) (keys 0-7, cols 8-15) (keys 8-15, cols 8-15)
                const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
                ldsm4_t(stage + C::HALF + row * (DP * 2) + swz(row, 2 * t + (lane >> 4)) * 16, r);
                mma16<T>(o[2 * t], p, r[0], r[1]);
                mma16<T>(o[2 * t + 1], p, r[2], r[3]);
            }
        }
    }
};

// The same for up to RR rows in fp32 by multiply-adds: a tensor-core tile would be mostly empty, and splitting K and V in two for it is
// what it spends its time on (16 sequences of up to 1100 keys, one row of each of 12 heads of 64: 38 us a call in tiles, 25 this way).  LPK
// lanes share a key, four values of it each; with width 64 the warp has two keys at a time.  Products and sums are plain fp32.
template <int DP, int RR> struct FewRows {
    using C = RowCfg<float, DP>;
    static constexpr int LPK = DP / 4, KPP = 32 / LPK, NP = C::CK / KPP, QR = RR * 4;

    float4 o[RR];
    float m[RR], l[RR];

    __device__ __forceinline__ static void load_q(const PagedArgs &a, const Unit &u, uint32_t (&qf)[QR]) {
        const int d = (int)(threadIdx.x % LPK) * 4;
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            const int row = u.rt * kRows + r, tok = row / a.group, hd = row - tok * a.group;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (tok < u.ql && d < a.dim)
                x = __ldg(reinterpret_cast<const uint4 *>((const float *)a.q + (long long)(u.t0 + tok) * a.q_tok + (long long)(u.h * a.group + hd) * a.q_head + d));
            qf[4 * r] = x.x, qf[4 * r + 1] = x.y, qf[4 * r + 2] = x.z, qf[4 * r + 3] = x.w;
        }
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int r = 0; r < RR; ++r)
            o[r] = make_float4(0.f, 0.f, 0.f, 0.f), m[r] = -INFINITY, l[r] = 0.f;
    }
    // Keys [base, base + CK) of a stage; row r sees keys below lim[r].
    __device__ __forceinline__ void step(const PagedArgs &a, const uint32_t (&qf)[QR], const unsigned char *stage, int base, const int (&lim)[RR], bool masked) {
        const int lane = threadIdx.x & 31, piece = lane % LPK, mine = lane / LPK;
        auto at = [&](int p) {
            const int row = p * KPP + mine;
            return row * (DP * 4) + RowTile<float, DP>::swz(row, piece) * 16;
        };
        float s[RR][NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const float4 k = *reinterpret_cast<const float4 *>(stage + at(p));
#pragma unroll
            for (int r = 0; r < RR; ++r) {
                float x = __uint_as_float(qf[4 * r]) * k.x;
                x = fmaf(__uint_as_float(qf[4 * r + 1]), k.y, x);
                x = fmaf(__uint_as_float(qf[4 * r + 2]), k.z, x);
                s[r][p] = fmaf(__uint_as_float(qf[4 * r + 3]), k.w, x);
            }
        }
#pragma unroll
        for (int w = LPK / 2; w > 0; w >>= 1)
#pragma unroll
            for (int r = 0; r < RR; ++r)
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    s[r][p] += __shfl_xor_sync(0xffffffffu, s[r][p], w);
        bool grows = false;
        float top[RR];
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                s[r][p] *= a.sl2;
                if (masked)
                    s[r][p] = base + p * KPP + mine < lim[r] ? s[r][p] : -INFINITY;
                top[r] = fmaxf(top[r], s[r][p]);
            }
            if (KPP > 1)
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], LPK & 31));
            grows |= top[r] > m[r];
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int r = 0; r < RR; ++r) {
                const float to = fmaxf(m[r], top[r]), f = m[r] == to ? 1.f : exp2_approx(m[r] - to);
                m[r] = to, l[r] *= f;
                o[r].x *= f, o[r].y *= f, o[r].z *= f, o[r].w *= f;
            }
        }
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            const float z = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                s[r][p] = exp2_approx(s[r][p] - z);
                l[r] += s[r][p];
            }
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const float4 v = *reinterpret_cast<const float4 *>(stage + C::HALF + at(p));
#pragma unroll
            for (int r = 0; r < RR; ++r)
                if (!masked || base + p * KPP + mine < lim[r]) // (0 times what a masked key holds could be NaN)
                    o[r].x = fmaf(s[r][p], v.x, o[r].x), o[r].y = fmaf(s[r][p], v.y, o[r].y), o[r].z = fmaf(s[r][p], v.z, o[r].z), o[r].w = fmaf(s[r][p], v.w, o[r].w);
        }
    }
    // The warp's sums where the block's warps meet; `seen[r]`: the row sees some of the warp's keys.
    __device__ __forceinline__ void leave(float *wo, float2 *wm, const bool (&seen)[RR]) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            if (KPP > 1) {
                o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, LPK & 31), o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, LPK & 31);
                o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, LPK & 31), o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, LPK & 31);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], LPK & 31);
            }
            if (lane < LPK)
                *reinterpret_cast<float4 *>(wo + r * C::MP + lane * 4) = o[r];
            if (lane == 0)
                wm[r] = make_float2(seen[r] ? fmaxf(m[r], -FLT_MAX) : -INFINITY, l[r]);
        }
    }
};

// What a piece's sums are scaled by beside the largest of all pieces' m.
__device__ __forceinline__ float piece_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2_approx(m - M); }

template <typename T> __device__ __forceinline__ void store4(T *p, float4 v) {
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(p) = v;
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}
// The row's result from its sums: zeros where it sees nothing.
__device__ __forceinline__ float4 settle(float4 v, float M, float L) {
    if (M == -INFINITY)
        return make_float4(0.f, 0.f, 0.f, 0.f);
    const float r = 1.f / L;
    return make_float4(v.x * r, v.y * r, v.z * r, v.w * r);
}
__device__ __forceinline__ void fma4(float4 &x, float w, float4 y) {
    x.x = fmaf(w, y.x, x.x), x.y = fmaf(w, y.y, x.y), x.z = fmaf(w, y.z, x.z), x.w = fmaf(w, y.w, x.w);
}

// FEW > 0 (fp32): no tile has more than that many rows.  most: of the sequences' steps (units where they are whole) there can be so many.
template <typename T, int DP, int FEW>
__global__ void __launch_bounds__(kRowThreads, RowCfg<T, DP>::CTAS) k_paged_rows(const PagedArgs a, int own_mode, unsigned most, int prefix_blocks, int prefix_pieces, int cluster) {
    using C = RowCfg<T, DP>;
    using Loader = RowTile<T, DP>;
    using Tile = typename std::conditional<FEW == 0, RowTile<T, DP>, FewRows<DP, FEW ? FEW : 1>>::type;
    pdl_prologue();
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ unsigned tmp[kRowWarps];
    __shared__ float2 joined[kRows]; // {m, l} of the block's rows, for its cluster
    __shared__ unsigned found[2]; // sequence that holds this CTA's first step, and where it begins
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    unsigned char *ring_p = smem + warp * C::WARP_BYTES;
    const uint32_t ring = ptx::smem_u32(ring_p);

    // ---- which steps are this CTA's ------------------------------------------------------------------------------
    // The first blocks take all tokens against the shared keys, as a single sequence without keys of its own: unit by unit, each in
    // pieces.  The others take the sequences.
    const bool one = (int)blockIdx.x < prefix_blocks;
    const int mode = one ? kModePieces : own_mode, seqs = one ? 1 : a.s.seqs, n0 = one || prefix_blocks == 0 ? a.s.n0 : 0;
    const unsigned grid = one ? prefix_blocks / prefix_pieces : gridDim.x - prefix_blocks;
    // (a unit's share of the cluster: all blocks of a cluster have one unit, and leave or stay together)
    const unsigned cta = one ? blockIdx.x / prefix_pieces : mode == kModeCluster ? blockIdx.x / cluster : blockIdx.x - prefix_blocks;
    const int rank = mode == kModeCluster ? (int)(blockIdx.x % cluster) : 0;
    const int piece = one ? (int)(blockIdx.x % prefix_pieces) : a.piece_out;
    auto visible = [&](int i, int n, int own) { return n0 + (a.causal ? min(max(own - n + i + 1, 0), own) : own); };
    auto tokens_of = [&](int b, int &t0) {
        if (one) {
            t0 = 0;
            return a.s.tokens;
        }
        return a.s.span(b, t0);
    };
    auto steps_of = [&](int b) { return mode == kModeRanges ? max(1, (n0 + a.s.own(b) + C::KT - 1) / C::KT) : 1; };
    auto cost_of = [&](int b) -> unsigned {
        int t0;
        const int tiles = ceil_div(tokens_of(b, t0) * a.group, kRows);
        return tiles ? (unsigned)(tiles * a.hkv) * (unsigned)steps_of(b) : 0u;
    };
    unsigned total = 0;
    for (int b0 = 0; b0 < seqs; b0 += kRowThreads) {
        unsigned t;
        block_scan(b0 + (int)threadIdx.x < seqs ? cost_of(b0 + threadIdx.x) : 0u, t, tmp);
        total = add_sat(total, t);
    }
    const unsigned G = mode == kModeRanges ? min(grid, total) : total;
    if (mode == kModeRanges && threadIdx.x == 0 && a.meta)
        a.meta[cta] = make_int4(-1, 0, 0, 0);
    if (a.s.q_starts && (int)blockIdx.x == prefix_blocks) { // (one block says so, of any excess; beyond `most` nothing is done)
        unsigned tokens = 0;
        for (int b0 = 0; b0 < seqs; b0 += kRowThreads) {
            unsigned t;
            int t0;
            block_scan(b0 + (int)threadIdx.x < seqs ? (unsigned)a.s.span(b0 + threadIdx.x, t0) : 0u, t, tmp);
            tokens = add_sat(tokens, t);
        }
        if (tokens > (unsigned)a.s.tokens && threadIdx.x == 0)
            atomicOr(a.s.status, kStatusStarts);
    }
    if (cta >= G || (!one && total > most))
        return;
    // whole units are taken from the last one down: later rows of a prompt see more keys
    const unsigned begin = mode == kModeRanges ? (unsigned)((unsigned long long)cta * total / G) : total - 1 - cta;
    const unsigned end = mode == kModeRanges ? (unsigned)((unsigned long long)(cta + 1) * total / G) : begin + 1;
    unsigned run = 0;
    for (int b0 = 0; b0 < seqs; b0 += kRowThreads) {
        unsigned t;
        const int b = b0 + threadIdx.x;
        const unsigned c = b < seqs ? cost_of(b) : 0u, at = run + block_scan(c, t, tmp);
        if (c && at <= begin && begin - at < c)
            found[0] = b, found[1] = at;
        run += t;
    }
    __syncthreads();
    int b = found[0];
    unsigned b_at = found[1];

    for (unsigned pos = begin; pos < end;) {
        unsigned c = cost_of(b);
        while (pos - b_at >= c) {
            b_at += c;
            c = cost_of(++b);
        }
        const unsigned steps = steps_of(b), unit = (pos - b_at) / steps, first = (pos - b_at) - unit * steps;
        const unsigned last = min(steps, first + (end - pos));
        Unit u;
        u.skip = a.s.n0 - n0;
        u.b = b, u.rt = unit / a.hkv, u.h = unit - u.rt * a.hkv;
        u.ql = tokens_of(b, u.t0);
        u.own = one ? 0 : a.s.own(b);
        const int row_end = min((u.rt + 1) * kRows, u.ql * a.group) - 1; // last row of the tile
        u.n = visible(row_end / a.group, u.ql, u.own);
        // the unit's steps of this CTA as keys
        const int all = (u.n + C::KT - 1) / C::KT;
        int s0 = first, s1 = min((int)last, all);
        if (mode == kModeUnits)
            s0 = 0, s1 = all;
        else if (mode == kModeCluster) {
            s0 = (int)((long long)all * rank / cluster), s1 = (int)((long long)all * (rank + 1) / cluster);
        } else if (mode == kModePieces) {
            s0 = (int)((long long)all * piece / prefix_pieces), s1 = (int)((long long)all * (piece + 1) / prefix_pieces);
        }
        const int r0 = u.rt * kRows + g, tok0 = r0 / a.group, tok1 = (r0 + 8) / a.group;
        const int lim0 = tok0 < u.ql ? visible(tok0, u.ql, u.own) : 0, lim1 = tok1 < u.ql ? visible(tok1, u.ql, u.own) : 0;
        const int full = visible(u.rt * kRows / a.group, u.ql, u.own); // keys that every row sees
        [[maybe_unused]] auto few_lim = [&](int r) {
            const int tok = (u.rt * kRows + r) / a.group;
            return tok < u.ql ? visible(tok, u.ql, u.own) : 0;
        };

        Tile tile;
        tile.reset();
        const int base0 = warp * C::CK;
#pragma unroll
        for (int st = 0; st < C::NST - 1; ++st) {
            const int key = (s0 + st) * C::KT + base0;
            if (s0 + st < s1 && key < u.n)
                Loader::fetch(a, u, ring + st * 2 * C::HALF, key, u.n);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        uint32_t qf[Tile::QR];
        Tile::load_q(a, u, qf);
        int st = 0;
#pragma unroll 1
        for (int i = s0; i < s1; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::NST - 2) : "memory");
            __syncwarp(); // every lane's copies of this stage are in, and every lane is done with the stage that is filled next
            {
                const int nx = i + C::NST - 1, key = nx * C::KT + base0, to = st == 0 ? C::NST - 1 : st - 1;
                if (nx < s1 && key < u.n)
                    Loader::fetch(a, u, ring + to * 2 * C::HALF, key, u.n);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
            const int key = i * C::KT + base0;
            if (key < u.n)
                if constexpr (FEW > 0) {
                    int lim[FEW];
#pragma unroll
                    for (int r = 0; r < FEW; ++r)
                        lim[r] = few_lim(r);
                    tile.step(a, qf, ring_p + st * 2 * C::HALF, key, lim, key + C::CK > full);
                } else
                    tile.step(a, qf, ring + st * 2 * C::HALF, ring_p + st * 2 * C::HALF, key, lim0, lim1, key + C::CK > full);
            st = st == C::NST - 1 ? 0 : st + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();

        // ---- the warps meet: {m, l} and O of each in its own stages --------------------------------------------------
        float *wo = reinterpret_cast<float *>(ring_p);
        float2 *wm = reinterpret_cast<float2 *>(wo + kRows * C::MP);
        if constexpr (FEW > 0) {
            bool seen[FEW];
#pragma unroll
            for (int r = 0; r < FEW; ++r)
                seen[r] = few_lim(r) > s0 * C::KT + base0 && s1 > s0; // this warp's first key at least
            tile.leave(wo, wm, seen);
        } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float l = tile.l[r];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int lim = r ? lim1 : lim0, seen = lim > s0 * C::KT + base0 && s1 > s0; // this warp's first key at least
                if ((lane & 3) == 0)
                    wm[g + 8 * r] = make_float2(seen ? fmaxf(tile.m[r], -FLT_MAX) : -INFINITY, l);
            }
            if constexpr (C::f32) {
#pragma unroll
                for (int t = 0; t < DP / 8; t += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<float4 *>(&wo[(g + 8 * (e >> 1)) * C::MP + Tile::column(t, e)]) =
                            make_float4(tile.o[t][e], tile.o[t + 1][e], tile.o[t + 2][e], tile.o[t + 3][e]);
            } else {
#pragma unroll
                for (int t = 0; t < DP / 8; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        *reinterpret_cast<float2 *>(&wo[(g + 8 * r) * C::MP + Tile::column(t, 0)]) = make_float2(tile.o[t][2 * r], tile.o[t][2 * r + 1]);
            }
        }
        __syncthreads();
        {
            const int row = threadIdx.x >> 3, part = threadIdx.x & 7, rg = u.rt * kRows + row, tok = rg / a.group, hd = rg - tok * a.group;
            if (tok < u.ql) {
                const bool whole = mode != kModeRanges || (first == 0 && last == steps);
                float M = -INFINITY, L = 0.f, w[kRowWarps];
#pragma unroll
                for (int x = 0; x < kRowWarps; ++x) {
                    w[x] = reinterpret_cast<const float2 *>(smem + x * C::WARP_BYTES + kRows * C::MP * 4)[row].x;
                    M = fmaxf(M, w[x]);
                }
#pragma unroll
                for (int x = 0; x < kRowWarps; ++x) {
                    w[x] = piece_weight(w[x], M);
                    L += w[x] * reinterpret_cast<const float2 *>(smem + x * C::WARP_BYTES + kRows * C::MP * 4)[row].y;
                }
                // To `out`; as a piece of the row; or, of a cut unit, as this block's first piece (continued from the block before) or
                // second (left to the one after); or to the cluster.
                float *po = nullptr;
                if (mode == kModeCluster) {
                } else if (!whole) {
                    const long long at = (long long)(2 * cta + (first > 0 ? 0 : 1)) * kRows + row;
                    po = a.ro + at * DP;
                    if (part == 0)
                        a.rml[at] = make_float2(M, L);
                } else if (piece >= 0) {
                    const long long at = ((long long)piece * a.hkv + u.h) * ((long long)a.s.tokens * a.group) + (long long)(u.t0 + tok) * a.group + hd;
                    po = a.po + at * DP;
                    if (part == 0)
                        a.pml[at] = make_float2(M, L);
                }
                T *out = (T *)a.out + (long long)(u.t0 + tok) * a.o_tok + (long long)(u.h * a.group + hd) * a.o_head;
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    const int col = j * 32 + part * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int x = 0; x < kRowWarps; ++x)
                        fma4(v, w[x], *reinterpret_cast<const float4 *>(smem + x * C::WARP_BYTES + (row * C::MP + col) * 4));
                    if (mode == kModeCluster) // (over the first warp's sums: nobody but this thread reads these)
                        *reinterpret_cast<float4 *>(smem + (row * C::MP + col) * 4) = v;
                    else if (po)
                        *reinterpret_cast<float4 *>(po + col) = v;
                    else if (col < a.dim)
                        store4<T>(out + col, settle(v, M, L));
                }
                if (mode == kModeCluster && part == 0)
                    joined[row] = make_float2(M, L);
            }
            if (mode == kModeCluster) {
                // The blocks of the cluster add their sums, each a share of the rows, from one another's shared memory.
                ptx::cluster_sync_all();
                constexpr int TPR = DP / 4; // threads of a row, four columns each
                for (int rr = rank + cluster * (int)(threadIdx.x / TPR); rr < kRows; rr += cluster * (kRowThreads / TPR)) {
                    const int rg2 = u.rt * kRows + rr, tok2 = rg2 / a.group, hd2 = rg2 - tok2 * a.group, col = (int)(threadIdx.x % TPR) * 4;
                    if (tok2 >= u.ql)
                        continue;
                    const uint32_t at_ml = ptx::smem_u32(&joined[rr]), at_o = ptx::smem_u32(smem + (rr * C::MP + col) * 4);
                    float M = -INFINITY, L = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int p = 0; p < cluster; ++p)
                        M = fmaxf(M, ptx::ld_dsmem_f32(ptx::map_to_cta(at_ml, p)));
#pragma unroll 4
                    for (int p = 0; p < cluster; ++p) {
                        const uint32_t m_at = ptx::map_to_cta(at_ml, p), o_at = ptx::map_to_cta(at_o, p);
                        const float f = piece_weight(ptx::ld_dsmem_f32(m_at), M);
                        L = fmaf(f, ptx::ld_dsmem_f32(m_at + 4), L);
                        fma4(v, f, make_float4(ptx::ld_dsmem_f32(o_at), ptx::ld_dsmem_f32(o_at + 4), ptx::ld_dsmem_f32(o_at + 8), ptx::ld_dsmem_f32(o_at + 12)));
                    }
                    if (col < a.dim)
                        store4<T>((T *)a.out + (long long)(u.t0 + tok2) * a.o_tok + (long long)(u.h * a.group + hd2) * a.o_head + col, settle(v, M, L));
                }
                ptx::cluster_sync_all(); // (a block's shared memory stays until the others have read it)
            }
            if (mode == kModeRanges && first > 0 && threadIdx.x == 0) {
                // The first CTA after the one in which the unit begins says where its pieces are.
                const unsigned from = pos - first, c0 = (unsigned)(((unsigned long long)(from + 1) * G - 1) / total);
                if (c0 + 1 == cta) {
                    const unsigned c1 = (unsigned)(((unsigned long long)(from + steps) * G - 1) / total);
                    a.meta[cta] = make_int4(u.b, u.rt, u.h, (int)c1);
                }
            }
        }
        __syncthreads(); // the stages are free again
        pos += last - first;
    }
}

// Sums of a row from n places, a pair of warps sharing them: lane l holds columns 4 l .. 4 l + 3, every second place is the other
// warp's.  `ml(i)` and `o(i)` say where place i lies.  The loads of eight places are in flight together, since what a row's pieces cost is
// trips to memory.  Answers in the first warp of the pair.
template <int DP, typename FM, typename FO> __device__ __forceinline__ void join_pair(int n, FM ml, FO o, float4 *tmp /*[4][32]*/, float (*tml)[2], float4 &v, float &M, float &L) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp & 1, pair = warp >> 1, col = DP == 128 ? lane * 4 : (lane & 15) * 4;
    M = -INFINITY, L = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 w[8];
    float4 x[8];
    auto load = [&](int i0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = min(i0 + 2 * e, n - 1);
            if (e < 1 || i0 + 2 * e < n) {
                w[e] = ml(i);
                x[e] = *reinterpret_cast<const float4 *>(o(i) + col);
            }
        }
    };
    if (half < n)
        load(half); // (with the maxima: the first sixteen places are one trip)
    for (int i = lane; i < n; i += 32)
        M = fmaxf(M, ml(i).x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
#pragma unroll 1
    for (int i0 = half; i0 < n; i0 += 16) {
        if (i0 != half)
            load(i0);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i0 + 2 * e < n) {
                const float f = piece_weight(w[e].x, M);
                L = fmaf(f, w[e].y, L);
                fma4(v, f, x[e]);
            }
    }
    if (half) {
        tmp[pair * 32 + lane] = v;
        tml[pair][0] = L;
    }
    __syncthreads();
    if (!half) {
        fma4(v, 1.f, tmp[pair * 32 + lane]);
        L += tml[pair][0];
    }
}

// Adds the pieces of the units that ranges have cut, four rows of a unit per CTA; CTA x looks after the unit that CTA x of the launch
// before found continued from CTA x - 1, where it began.
template <typename T, int DP> __global__ void __launch_bounds__(256) k_paged_join(const PagedArgs a) {
    pdl_prologue();
    __shared__ float4 tmp[4 * 32];
    __shared__ float tml[4][2];
    const int4 d = a.meta[blockIdx.x];
    if (d.x < 0)
        return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 4 + (warp >> 1);
    int t0;
    const int ql = a.s.span(d.x, t0), rg = d.y * kRows + row, tok = rg / a.group, hd = rg - tok * a.group;
    const int c0 = (int)blockIdx.x - 1, n = tok < ql ? d.w - c0 + 1 : 0;
    // (the unit is the second piece of the CTA that it begins in, and the first of the others)
    auto place = [&](int i) { return (long long)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * kRows + row; };
    float4 v;
    float M, L;
    join_pair<DP>(n, [&](int i) { return a.rml[place(i)]; }, [&](int i) { return a.ro + place(i) * DP; }, tmp, tml, v, M, L);
    const int col = lane * 4;
    if ((warp & 1) || n == 0 || col >= DP)
        return;
    if (a.piece_out >= 0) {
        const long long at = ((long long)a.piece_out * a.hkv + d.z) * ((long long)a.s.tokens * a.group) + (long long)(t0 + tok) * a.group + hd;
        *reinterpret_cast<float4 *>(a.po + at * DP + col) = v;
        if (lane == 0)
            a.pml[at] = make_float2(M, L);
    } else if (col < a.dim)
        store4<T>((T *)a.out + (long long)(t0 + tok) * a.o_tok + (long long)(d.z * a.group + hd) * a.o_head + col, settle(v, M, L));
}

// Adds the pieces of every row, four (token, head) pairs per CTA.
template <typename T, int DP> __global__ void __launch_bounds__(256) k_paged_join_rows(const PagedArgs a) {
    pdl_prologue();
    __shared__ float4 tmp[4 * 32];
    __shared__ float tml[4][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.hkv * a.group;
    const long long rows = (long long)a.s.tokens * a.group, id = (long long)blockIdx.x * 4 + (warp >> 1);
    const int tok = (int)(id / heads), head = (int)(id - (long long)tok * heads), h = head / a.group;
    int n = id < rows * a.hkv ? a.pieces : 0;
    if (n && a.s.q_starts && (tok < __ldg(a.s.q_starts) || tok >= __ldg(a.s.q_starts + a.s.seqs)))
        n = 0; // rows outside all sequences stay as they were
    auto place = [&](int p) { return ((long long)p * a.hkv + h) * rows + (long long)tok * a.group + (head - h * a.group); };
    float4 v;
    float M, L;
    join_pair<DP>(n, [&](int i) { return a.pml[place(i)]; }, [&](int i) { return a.po + place(i) * DP; }, tmp, tml, v, M, L);
    const int col = lane * 4;
    if (!(warp & 1) && n && col < a.dim)
        store4<T>((T *)a.out + (long long)tok * a.o_tok + (long long)head * a.o_head + col, settle(v, M, L));
}

// The same for up to four pieces: a warp per row, all that it reads in one trip, and registers for eight blocks an SM instead of two
// (11 k rows of two pieces: 19 us with the pairs of warps above).
template <typename T, int DP> __global__ void __launch_bounds__(256) k_paged_join_four(const PagedArgs a) {
    pdl_prologue();
    const int lane = threadIdx.x & 31, heads = a.hkv * a.group, col = DP == 128 ? lane * 4 : (lane & 15) * 4;
    const long long rows = (long long)a.s.tokens * a.group, id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= rows * a.hkv)
        return;
    const int tok = (int)(id / heads), head = (int)(id - (long long)tok * heads), h = head / a.group;
    const int first = a.s.q_starts ? __ldg(a.s.q_starts) : 0, last = a.s.q_starts ? __ldg(a.s.q_starts + a.s.seqs) : a.s.tokens;
    float2 ml[4];
    float4 x[4];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        ml[p] = make_float2(-INFINITY, 0.f);
        x[p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < a.pieces) {
            const long long at = ((long long)p * a.hkv + h) * rows + (long long)tok * a.group + (head - h * a.group);
            ml[p] = a.pml[at];
            x[p] = *reinterpret_cast<const float4 *>(a.po + at * DP + col);
        }
    }
#pragma unroll
    for (int p = 0; p < 4; ++p)
        M = fmaxf(M, ml[p].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float f = piece_weight(ml[p].x, M);
        L = fmaf(f, ml[p].y, L);
        fma4(v, f, x[p]);
    }
    if (tok >= first && tok < last && lane * 4 < a.dim) // (rows outside all sequences stay as they were)
        store4<T>((T *)a.out + (long long)tok * a.o_tok + (long long)head * a.o_head + col, settle(v, M, L));
}

template <typename T, int DP, int FEW>
int rows_launch_as(petb200_ctx *ctx, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int n_prefix, cudaStream_t s) {
    using C = RowCfg<T, DP>;
    const long long rows = (long long)a.s.tokens * a.group;
    // Row tiles there can be: a sequence's last one may be short.
    const long long tiles = a.s.q_starts ? rows / kRows + a.s.seqs : a.s.seqs * (((long long)a.s.q_len * a.group + kRows - 1) / kRows);
    const long long units = tiles * a.hkv, own = (long long)a.s.width * a.s.page_size, keys = own + (n_prefix ? 0 : a.s.n0);
    const long long steps = std::max(1ll, (keys + C::KT - 1) / C::KT), prefix_blocks = (rows + kRows - 1) / kRows * a.hkv * n_prefix;
    if (own + a.s.n0 > 0x7fff0000ll || units * steps + prefix_blocks > 0x7fff0000ll || rows > 0x7fff0000ll)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "attention over pages: %lld row tiles of up to %lld keys are more than one call takes", units, keys);
    const int slots = ctx->sm_count * C::CTAS;
    // Units as they are where there are several rounds of them (ranges would cut each in two for a gain of a part of a round), or
    // where a unit is a few steps (a second launch would cost more than they).  Two rounds do where units are short: 1024 units of up to
    // 500 keys behind a prefix 96 us for the call, 114 with ranges; units of thousands of keys lose 7 % that way.
    // Few units of moderate length go to a cluster of blocks each, which add their sums through shared memory: one launch and no
    // workspace (one token on 1500 keys, 8 units: 15.5 us a call with ranges, whose second launch alone costs the host 2.5).
    const int cluster = n_prefix || a.piece_out >= 0 || steps <= 4 ? 0 : units * 8 <= slots && steps <= 64 ? 8 : units * 4 <= slots && steps <= 32 ? 4 : 0;
    const int mode = cluster ? kModeCluster : units >= (steps <= 16 ? 2ll : 4ll) * slots || steps <= 4 ? kModeUnits : kModeRanges;
    const unsigned grid = (unsigned)(mode == kModeRanges ? std::min<long long>(slots, units * steps) : mode == kModeCluster ? units * cluster : units);
    size_t bytes = 0;
    if (mode == kModeRanges) {
        a.ro = reinterpret_cast<float *>(ws);
        bytes = (size_t)grid * 2 * kRows * DP * 4;
        a.rml = reinterpret_cast<float2 *>(ws + bytes);
        bytes += (size_t)grid * 2 * kRows * 8;
        a.meta = reinterpret_cast<int4 *>(ws + bytes);
        bytes += (size_t)grid * 16;
    }
    *need = bytes;
    if (!a.q) // (asked for the size alone)
        return PETB200_OK;
    if (bytes > ws_bytes)
        return fail(ctx, PETB200_ERR_INVALID, "attention over pages: a workspace of %zu bytes, %zu are needed", ws_bytes, bytes);
    if (int rc = raise_smem(ctx, (const void *)k_paged_rows<T, DP, FEW>, C::SMEM))
        return rc;
    if (mode == kModeCluster) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(grid), cfg.blockDim = dim3(kRowThreads), cfg.dynamicSmemBytes = C::SMEM, cfg.stream = s;
        cudaLaunchAttribute attr[2]{};
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr, cfg.numAttrs = pdl_enabled() ? 2 : 1;
        (void)cudaLaunchKernelEx(&cfg, k_paged_rows<T, DP, FEW>, a, mode, (unsigned)units, 0, 1, cluster);
        return launched(ctx, "k_paged_rows");
    }
    launch_pdl(k_paged_rows<T, DP, FEW>, dim3(grid + (unsigned)prefix_blocks), kRowThreads, C::SMEM, s, a, mode,
               (unsigned)(mode == kModeRanges ? units * steps : units), (int)prefix_blocks, std::max(1, n_prefix), 1);
    int rc = launched(ctx, "k_paged_rows");
    if (rc || mode != kModeRanges)
        return rc;
    // (an even call's tiles have no more rows than its sequences)
    const int four = (int)std::min<long long>(kRows / 4, a.s.q_starts ? kRows / 4 : ((long long)a.s.q_len * a.group + 3) / 4);
    launch_pdl(k_paged_join<T, DP>, dim3(grid, (unsigned)four), 256, 0, s, a);
    return launched(ctx, "k_paged_join");
}

template <typename T, int DP>
int rows_launch(petb200_ctx *ctx, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int n_prefix, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) { // (the prefix's tiles have other sequences' rows in them)
        const long long rows = a.s.q_starts || n_prefix ? kRows : (long long)a.s.q_len * a.group;
        if (rows == 1)
            return rows_launch_as<T, DP, 1>(ctx, a, ws, ws_bytes, need, n_prefix, s);
        if (rows <= 4)
            return rows_launch_as<T, DP, 4>(ctx, a, ws, ws_bytes, need, n_prefix, s);
    }
    return rows_launch_as<T, DP, 0>(ctx, a, ws, ws_bytes, need, n_prefix, s);
}

template <typename T, int DP> int join_launch(petb200_ctx *ctx, const PagedArgs &a, cudaStream_t s) {
    const long long rows = (long long)a.s.tokens * a.group * a.hkv;
    if (a.pieces <= 4) {
        launch_pdl(k_paged_join_four<T, DP>, dim3((unsigned)((rows + 7) / 8)), 256, 0, s, a);
        return launched(ctx, "k_paged_join_four");
    }
    launch_pdl(k_paged_join_rows<T, DP>, dim3((unsigned)((rows + 3) / 4)), 256, 0, s, a);
    return launched(ctx, "k_paged_join_rows");
}

} // namespace

int paged_rows_run(petb200_ctx *ctx, int dtype, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int n_prefix, cudaStream_t s) {
    const bool wide = a.dim > 64;
    switch (dtype) {
    case PETB200_F16:
        return wide ? rows_launch<__half, 128>(ctx, a, ws, ws_bytes, need, n_prefix, s) : rows_launch<__half, 64>(ctx, a, ws, ws_bytes, need, n_prefix, s);
    case PETB200_BF16:
        return wide ? rows_launch<__nv_bfloat16, 128>(ctx, a, ws, ws_bytes, need, n_prefix, s)
                    : rows_launch<__nv_bfloat16, 64>(ctx, a, ws, ws_bytes, need, n_prefix, s);
    default:
        return wide ? rows_launch<float, 128>(ctx, a, ws, ws_bytes, need, n_prefix, s) : rows_launch<float, 64>(ctx, a, ws, ws_bytes, need, n_prefix, s);
    }
}

int paged_join_rows(petb200_ctx *ctx, int dtype, const PagedArgs &a, cudaStream_t s) {
    const bool wide = a.dim > 64;
    switch (dtype) {
    case PETB200_F16:
        return wide ? join_launch<__half, 128>(ctx, a, s) : join_launch<__half, 64>(ctx, a, s);
    case PETB200_BF16:
        return wide ? join_launch<__nv_bfloat16, 128>(ctx, a, s) : join_launch<__nv_bfloat16, 64>(ctx, a, s);
    default:
        return wide ? join_launch<float, 128>(ctx, a, s) : join_launch<float, 64>(ctx, a, s);
    }
}

} // namespace petb200
