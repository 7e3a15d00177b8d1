// Attention of many query rows over a paged cache on the fifth-generation tensor cores (16-bit types): prompts, pieces of prompts,
// and the shared prefix of a batch.
//
//   S = Q K^T,  P = 2^(S scale log2(e) - m),  O = sum P V,  out = O / l        (m, l: running maximum and sum of a row, fp32)
//
// A unit is 256 rows = (token, query head) pairs that share one key head, as two tiles of 128, against 128 keys at a time.  TMEM holds
// both tiles' scores (fp32) and outputs, all 512 columns at head width 128; P takes its scores' place as 16-bit values and is the A operand
// of the second product from there.  Roles: warps 0-3 and 4-7 do the softmax of a tile each (a thread owns a row), warps 8-11 fetch
// (warp 10 the keys, the others first the queries), warp 15 issues the products.  The products of one tile run under the softmax of
// the other.
//   tensor pipe  2 x (S: 128 x 128 x D, O: 128 x D x 128) = 2048 cycles per 128 keys at D = 128
//   exponentials 2 x 16384 at 16 a cycle                  = 2048 cycles
// Measured at D = 128: 3360 cycles per 128 keys.  What bounds it is the chain of one tile: its softmax (1800 cycles: 220 for reading the
// scores, 320 for the maximum, 1280 for the powers, whose 450 instructions come at three cycles each), the hand-over (350) and its
// two products (1270).  Tried and no faster: part of the powers as polynomials on the FMA pipe (more instructions), two threads a row,
// quarters of a tile in a rolled loop, the maximum of the tile before taken first and checked beside the powers, and blocks that
// stay and take unit after unit (registers spilled).  Beside the keys a unit costs 11 k cycles until its first scores and 5 k for its
// results.  500 tokens x 16 heads on 33 k keys: 149 to 151 us, 890 TFLOP/s; tensor pipe busy 58 % (profiles/paged_attention.md).
// The maximum moves only where a row's grows by more than 2^8 over the one in use (then O and l are scaled, by the softmax warps): the
// sums stay within range and any m gives the same quotient.  fp16 takes the maximum less 7 (see lifted()).
//
// K and V tiles are fetched by TMA, a box per page (or part of a page) and 64 columns, in the 128-byte swizzle (16-byte piece c of row r at
// c ^ (r & 7)); V is the second product's B operand as it lies, its rows along K ("MN-major").  Pages that do not fit the tiles (a
// page size that neither divides 128 nor is a multiple of it, or is below 8) come by 16-byte asynchronous copies of four warps
// instead, which is issue-bound: 5.1 k cycles per 128 keys.  Keys count in tiles from the first shared key and again from the first own
// key, so that a tile never straddles the two.
//
// A masked key's score is replaced before the maximum.  Rows of V that no row of the unit sees are zeros in shared memory, whatever
// the page holds there.  Where some row of the unit does not see some key of a tile, the fetching warps look for non-finite values of
// V and take them out (0 x infinity would be NaN); the rows that do see them get them back at the end.
#include "paged.cuh"
#include "tc_ptx.cuh"
#include <algorithm>
#include <cfloat>

namespace petb200 {
namespace {

constexpr int kTileRows = 128, kTileKeys = 128, kTileThreads = 512;
constexpr int kSoftmaxRegs = 176, kOtherRegs = 80;
static_assert(256 * (kSoftmaxRegs + kOtherRegs) <= kTileThreads * 128, "more registers than the block was launched with: setmaxnreg would wait forever");
constexpr int kLag = 2; // stages whose copies a fetching thread leaves in flight before it reports the one before them
constexpr float kGrowth = 8.f;

template <int DP> struct TileCfg {
    static constexpr int STAGE = kTileKeys * DP * 2;
    static constexpr int NS = DP == 128 ? 5 : 8; // stages of the ring, K and V in turn
    static constexpr int Q = 2 * kTileRows * DP * 2;
    static constexpr int SMEM = Q + NS * STAGE + 2048 + 512; // tiles (at the block's base, which is 1024-byte aligned), row table, control
    static constexpr int SUBS = DP / 64;         // blocks of 64 columns (128 bytes) of a tile
    static constexpr int CPR = DP / 8, RP = 128 / CPR, NP = 128 / RP; // pieces of a row; rows of a pass of the 128 threads; passes
};
static_assert(TileCfg<128>::SMEM <= 227 * 1024, "shared memory of a block");

struct TileCtl {
    uint64_t q_full, raw, full[8], empty[8], s_full[2], p_full[2][2], o_full[2]; // raw: a V tile that is looked over before it is full
    uint32_t tmem;
    int abort, bad; // bad: non-finite values of V were taken out
    int b, unit;
};
static_assert(sizeof(TileCtl) <= 512, "control block");

// Barrier among `threads` threads that answers whether `v` held for all of them.
__device__ __forceinline__ bool named_bar_all(int id, int threads, bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\tbar.red.and.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(r) : "r"(id), "r"(threads), "r"((uint32_t)v) : "memory");
    return r != 0;
}

// D[tmem] (+)= A[smem] * B[smem], 16-bit inputs, fp32 accumulate; one thread issues.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// Operand whose rows lie along K, 64 values (128 bytes) of the other extent each, in the 128-byte swizzle: blocks of 64 values are
// `block` bytes apart, groups of eight rows 1024.
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t smem_addr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3ffff) >> 4);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
constexpr uint32_t kIdescBMajorMN = 1u << 16;

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value)
        return ptx::pack_f16x2(a, b);
    else
        return ptx::pack_bf16x2(a, b);
}
// 0 * w + c of two 16-bit values: a zero stays one unless a value is not finite
template <typename T> __device__ __forceinline__ uint32_t zero_times(uint32_t w, uint32_t c) {
    uint32_t d;
    if constexpr (std::is_same<T, __half>::value)
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(c));
    else
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(c));
    return d;
}
// Values whose exponent bits are all set, taken out
template <typename T> __device__ __forceinline__ uint32_t word_clean(uint32_t w) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return ((w & e) == e ? 0u : w & 0xffffu) | (((w >> 16) & e) == e ? 0u : w & 0xffff0000u);
}

template <typename T, int DP> __global__ void __launch_bounds__(kTileThreads, 1)
    k_paged_tiles(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PagedArgs a, int splits, int to_pieces, int tma, int starve) {
    using C = TileCfg<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    int2 *row_table = reinterpret_cast<int2 *>(smem + C::Q + C::NS * C::STAGE); // [2][128]: a tile's keys as {page (-1: zeros), slot}
    TileCtl &ctl = *reinterpret_cast<TileCtl *>(smem + C::Q + C::NS * C::STAGE + 2048);
    const uint32_t q_s = ptx::smem_u32(smem), ring = q_s + C::Q;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort_flag = &ctl.abort;
    if (q_s & 1023) { // (the swizzle counts from 1024-byte boundaries; a block's dynamic memory begins on one)
        if (threadIdx.x == 0)
            atomicOr(a.s.status, kStatusWait);
        return;
    }

    if (threadIdx.x == 0) {
        ptx::mbar_init(&ctl.q_full, tma ? 96 : 128);
        ptx::mbar_init(&ctl.raw, 1);
        for (int i = 0; i < C::NS; ++i) {
            ptx::mbar_init(&ctl.full[i], (tma ? 1 : 128) + starve); // (starve, a test hook: an arrival that never comes)
            ptx::mbar_init(&ctl.empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(&ctl.s_full[t], 1);
            ptx::mbar_init(&ctl.p_full[t][0], 128);
            ptx::mbar_init(&ctl.p_full[t][1], 128);
            ptx::mbar_init(&ctl.o_full[t], 1);
        }
        ctl.abort = ctl.bad = 0;
        ctl.b = -1;
        ptx::fence_mbar_init();
    }
    if (warp == 15) {
        ptx::tmem_alloc(&ctl.tmem, 512);
        ptx::tmem_relinquish();
    }
    // A kernel that follows may start once every block of this one has come here: all that ran before this kernel is then done, and
    // it may read what that wrote without waiting for this kernel.
    ptx::grid_dep_wait();
    ptx::grid_dep_launch_dependents();
    __syncthreads();

    // ---- which unit, which keys --------------------------------------------------------------------------------------------
    const bool one = a.s.kv_lens == nullptr; // all tokens against the shared keys: a single sequence without keys of its own
    auto tokens_of = [&](int b, int &t0) {
        if (one) {
            t0 = 0;
            return a.s.tokens;
        }
        return a.s.span(b, t0);
    };
    auto units_of = [&](int b) {
        int t0;
        return ceil_div(tokens_of(b, t0) * a.group, 2 * kTileRows) * a.hkv;
    };
    const int split = blockIdx.x % splits, place = blockIdx.x / splits;
    if (warp == 0) { // units are laid end to end and taken from the last one down: later rows of a prompt see more keys
        const int seqs = one ? 1 : a.s.seqs;
        auto count = [&](int b0) { return !one && a.s.q_starts && b0 + lane < seqs ? (unsigned)units_of(b0 + lane) : 0u; };
        unsigned c = count(0), total = c;
#pragma unroll 4
        for (int b0 = 32; b0 < seqs; b0 += 32)
            total += count(b0);
        total = __reduce_add_sync(0xffffffffu, total);
        if (one || !a.s.q_starts) { // as many of each
            const unsigned per = (unsigned)units_of(0), all = per * (unsigned)seqs;
            if ((unsigned)place < all)
                ctl.b = (int)((all - 1 - place) / per), ctl.unit = (int)((all - 1 - place) % per);
        } else if ((unsigned)place < total) {
            const unsigned mine = total - 1 - place;
            unsigned run = 0;
            for (int b0 = 0; b0 < seqs && run <= mine; b0 += 32) {
                if (b0 > 0)
                    c = count(b0);
                unsigned inc = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
                    inc += lane >= o ? v : 0u;
                }
                const unsigned at = run + inc - c;
                if (c && at <= mine && mine - at < c)
                    ctl.b = b0 + lane, ctl.unit = (int)(mine - at);
                run += __shfl_sync(0xffffffffu, inc, 31);
            }
        }
    }
    if (warp == 12 && blockIdx.x == 0 && !one && a.s.q_starts) { // (one block says that the starts run backwards)
        unsigned long long tokens = 0;
        for (int b0 = lane, t0; b0 < a.s.seqs; b0 += 32)
            tokens += (unsigned)a.s.span(b0, t0);
        for (int o = 16; o > 0; o >>= 1)
            tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
        if (tokens > (unsigned long long)a.s.tokens && lane == 0)
            atomicOr(a.s.status, kStatusStarts);
    }
    __syncthreads();
    const uint32_t tmem = ctl.tmem;
    const int b = ctl.b;
    if (b >= 0) {
        const int rt = ctl.unit / a.hkv, h = ctl.unit - rt * a.hkv, row0 = rt * 2 * kTileRows;
        int t0;
        const int ql = tokens_of(b, t0), own = one ? 0 : a.s.own(b), rows = min(2 * kTileRows, ql * a.group - row0);
        const int tiles = rows > kTileRows ? 2 : 1;
        // own keys that the last row sees, and the first; the rows see all shared keys
        const int n0 = a.s.n0, own_last = a.s.visible((row0 + rows - 1) / a.group, ql, own, a.causal) - n0;
        const int own_first = a.s.visible(row0 / a.group, ql, own, a.causal) - n0;
        const int tiles0 = (n0 + kTileKeys - 1) / kTileKeys, all = tiles0 + (own_last + kTileKeys - 1) / kTileKeys;
        const int k0 = (int)((long long)all * split / splits), k1 = (int)((long long)all * (split + 1) / splits), steps = k1 - k0;
        // A tile's first key (counted in its part), its part's end, and the key of the whole sequence that its first is
        auto first_key = [&](int j) { return (j < tiles0 ? j : j - tiles0) * kTileKeys; };
        auto part_end = [&](int j) { return j < tiles0 ? n0 : own_last; };
        auto whole_key = [&](int j) { return first_key(j) + (j < tiles0 ? 0 : n0); };

        if (warp >= 8 && warp < 12) {
            ptx::reg_dealloc<kOtherRegs>();
            // ---- fetch ------------------------------------------------------------------------------------------------
            const int lt = threadIdx.x - 256, piece = lt % C::CPR, r0 = lt / C::CPR;
            const uint32_t at0 = (uint32_t)((piece >> 3) * (kTileKeys * 128) + r0 * 128 + (((piece & 7) ^ (r0 & 7)) << 4)); // (rows of a thread agree in r & 7)
            const bool col = piece * 8 < a.dim;
            const T *kc = (const T *)a.kc + (long long)h * a.kh + piece * 8, *vc = (const T *)a.vc + (long long)h * a.vh + piece * 8;
            // The query rows, by `count` threads of which this is the `me`-th.  Where each row lies is worked out once, by one of them.
            auto fetch_q = [&](int me, int count) {
                long long *where = reinterpret_cast<long long *>(row_table);
#pragma unroll 1
                for (int r = me; r < tiles * kTileRows; r += count) {
                    const int tok = (row0 + r) / a.group, hd = row0 + r - tok * a.group;
                    where[r] = r < rows ? (long long)(t0 + tok) * a.q_tok + (long long)(h * a.group + hd) * a.q_head : -1;
                }
                ptx::named_bar_sync(2, count);
#pragma unroll 4
                for (int i = me; i < tiles * kTileRows * C::CPR; i += count) {
                    const int r = i / C::CPR, c = i % C::CPR;
                    const long long at = where[r];
                    const bool in = c * 8 < a.dim && at >= 0;
                    cp_async_16_or_zero(q_s + (r >> 7) * (C::Q / 2) + (c >> 3) * (kTileRows * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
                                        (const T *)a.q + (in ? at + c * 8 : 0), in ? 16 : 0);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            // Looks over this thread's pieces of the V tile in stage `st`: rows past the part's end become zeros, non-finite values too
            // where some row does not see some key of the tile (among shared keys every row sees all).
            auto scrub = [&](int j, int st) {
                unsigned char *p = smem + C::Q + st * C::STAGE + at0;
                const int left = part_end(j) - first_key(j);
                if (left < kTileKeys)
#pragma unroll 1
                    for (int i = 0; i < C::NP; ++i)
                        if (i * C::RP + r0 >= left)
                            *reinterpret_cast<uint4 *>(p + i * (C::RP * 128)) = make_uint4(0u, 0u, 0u, 0u);
                if (j < tiles0)
                    return;
                uint32_t any = 0; // pairs of zeros, or of what 0 x infinity and 0 x NaN give
#pragma unroll 4
                for (int i = 0; i < C::NP; ++i) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(p + i * (C::RP * 128));
                    any = zero_times<T>(x.w, zero_times<T>(x.z, zero_times<T>(x.y, zero_times<T>(x.x, any))));
                }
                if ((any & 0x7fff7fffu) == 0)
                    return;
#pragma unroll 1
                for (int i = 0; i < C::NP; ++i) {
                    uint4 *w = reinterpret_cast<uint4 *>(p + i * (C::RP * 128));
                    const uint4 x = *w;
                    *w = make_uint4(word_clean<T>(x.x), word_clean<T>(x.y), word_clean<T>(x.z), word_clean<T>(x.w));
                }
                *(volatile int *)&ctl.bad = 1;
            };
            auto partly = [&](int j) { return first_key(j) + kTileKeys > (j < tiles0 ? n0 : own_first); };
            if (tma) {
                if (warp != 10 && steps > 0) { // (one warp goes ahead with the keys)
                    fetch_q(warp < 10 ? lt : lt - 32, 96);
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(&ctl.q_full);
                }
                const int box = min(a.s.page_size, kTileKeys), boxes = kTileKeys / box, sub = lane % C::SUBS, mine = lane / C::SUBS;
                // A lane looks up the page of its box, a tile ahead.  No page (past the keys, or not one): a page past the last, zeros.
                int page = 0, slot = 0;
                auto look = [&](int j) {
                    const int key = first_key(j) + mine * box;
                    page = a.s.pages;
                    if (mine < boxes && key < part_end(j)) {
                        page = a.s.entry(b, whole_key(j) + mine * box, slot);
                        if (!a.s.is_page(page)) {
                            atomicOr(a.s.status, kStatusPage);
                            page = a.s.pages;
                        }
                    }
                };
                if (warp == 10 && steps > 0)
                    look(k0);
                bool ok = true;
                int looked = 0; // V tiles looked over so far
                for (int j = k0; j < k1; ++j) {
                    const bool over = partly(j);
                    const int iv = 2 * (j - k0) + 1, sv = iv % C::NS;
                    if (warp == 10) {
                        const int p = page, sl = slot;
                        if (j + 1 < k1)
                            look(j + 1);
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const int item = 2 * (j - k0) + v, st = item % C::NS, use = item / C::NS;
                            if (use > 0)
                                ok = ok && ptx::mbar_wait_warp(&ctl.empty[st], (use - 1) & 1, abort_flag);
                            if (ok) {
                                uint64_t *bar = v && over ? &ctl.raw : &ctl.full[st];
                                if (lane == 0)
                                    ptx::mbar_expect_tx(bar, C::STAGE);
                                __syncwarp();
                                if (mine < boxes)
                                    ptx::tma_load_4d(smem + C::Q + st * C::STAGE + sub * (kTileKeys * 128) + mine * box * 128, v ? &vmap : &kmap, bar, sub * 64, sl, h, p);
                            }
                        }
                    } else if (!over)
                        continue;
                    if (over) { // (warps 9 to 11 come here for these tiles alone, in step with warp 8)
                        ok = named_bar_all(1, 128, ok);
                        if (!ok)
                            break;
                        ok = ptx::mbar_wait(&ctl.raw, looked++ & 1, abort_flag);
                        if (ok)
                            scrub(j, sv);
                        ptx::fence_proxy_async_smem();
                        ok = named_bar_all(1, 128, ok);
                        if (!ok)
                            break;
                        if (lt == 0)
                            ptx::mbar_arrive(&ctl.full[sv]);
                    }
                }
            } else {
                if (steps > 0) {
                    fetch_q(lt, 128);
                    ptx::named_bar_sync(1, 128); // (the row table is free)
                }
                int issued = steps > 0 ? 1 : 0, told = 0; // of Q, K 0, V 0, K 1, ...
                auto tell = [&]() {                      // the oldest of them has arrived: its own copies, then everyone's
                    if (told > 0 && !(told & 1)) {
                        const int j = k0 + told / 2 - 1;
                        if (partly(j))
                            scrub(j, (told - 1) % C::NS);
                    }
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(told == 0 ? &ctl.q_full : &ctl.full[(told - 1) % C::NS]);
                    ++told;
                };
                // A thread looks up one key of the tile, a tile ahead, and leaves it in the row table; the copies read the places there.
                int page = 0, slot = 0;
                auto look = [&](int j) {
                    if (first_key(j) + lt < part_end(j))
                        page = a.s.entry(b, whole_key(j) + lt, slot);
                };
                bool ok = true;
                if (steps > 0)
                    look(k0);
                for (int j = k0; j < k1; ++j) {
                    int2 *rows_j = row_table + (j & 1) * kTileKeys;
                    const bool in = first_key(j) + lt < part_end(j), is_page = a.s.is_page(page);
                    if (in && !is_page)
                        atomicOr(a.s.status, kStatusPage);
                    rows_j[lt] = make_int2(in && is_page ? page : -1, slot);
                    if (j + 1 < k1)
                        look(j + 1);
                    ok = named_bar_all(1, 128, ok); // (all of them leave together)
                    if (!ok)
                        break;
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int item = issued - 1, s = item % C::NS, use = item / C::NS;
                        if (use > 0 && !ptx::mbar_try_wait(&ctl.empty[s], (use - 1) & 1)) {
                            asm volatile("cp.async.wait_group 0;" ::: "memory"); // whoever empties the stage may be waiting for these
                            while (told < issued)
                                tell();
                            ok = ok && ptx::mbar_wait(&ctl.empty[s], (use - 1) & 1, abort_flag);
                        }
                        if (ok) {
                            const uint32_t dst = ring + s * C::STAGE + at0;
                            const T *base = v ? vc : kc;
                            const long long sp = v ? a.vp : a.kp, ss = v ? a.vs : a.ks;
                            // (places of eight rows are read before their copies: a copy's asm keeps later reads behind it)
#pragma unroll
                            for (int i0 = 0; i0 < C::NP; i0 += 8) {
                                const T *src[8];
                                int bytes[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const int2 at = rows_j[(i0 + i) * C::RP + r0];
                                    bytes[i] = col && at.x >= 0 ? 16 : 0;
                                    src[i] = base + (bytes[i] ? (long long)at.x * sp + (long long)at.y * ss : 0);
                                }
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    cp_async_16_or_zero(dst + (i0 + i) * (C::RP * 128), src[i], bytes[i]);
                            }
                            asm volatile("cp.async.commit_group;" ::: "memory");
                            ++issued;
                            if (issued - told > kLag) {
                                asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                                tell();
                            }
                        }
                    }
                }
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                while (told < issued)
                    tell();
            }
        } else if (warp >= 12) {
            ptx::reg_dealloc<kOtherRegs>();
            // ---- products ------------------------------------------------------------------------------------------------
            if (warp == 15 && steps > 0 && ptx::elect_one()) {
                const uint32_t kind = std::is_same<T, __half>::value ? ptx::idesc_f16(kTileRows, kTileKeys) : ptx::idesc_bf16(kTileRows, kTileKeys);
                const uint32_t kind_o = (std::is_same<T, __half>::value ? ptx::idesc_f16(kTileRows, DP) : ptx::idesc_bf16(kTileRows, DP)) | kIdescBMajorMN;
                auto scores = [&](int t, int s) {
                    const uint64_t qa = ptx::smem_desc_k128(q_s + t * (C::Q / 2)), kb = ptx::smem_desc_k128(ring + s * C::STAGE);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) { // (addresses count in 16 bytes)
                        const uint64_t off = ((k >> 2) * (kTileKeys * 128) + (k & 3) * 32) >> 4;
                        mma_f16_ss(tmem + t * 128, qa + off, kb + off, kind, k > 0);
                    }
                    ptx::mma_commit(&ctl.s_full[t]);
                };
                bool ok = ptx::mbar_wait(&ctl.q_full, 0, abort_flag) && ptx::mbar_wait(&ctl.full[0], 0, abort_flag);
                if (ok) {
                    ptx::tc_fence_after();
                    for (int t = 0; t < tiles; ++t)
                        scores(t, 0);
                    ptx::mma_commit(&ctl.empty[0]);
                }
                for (int j = 0; j < steps && ok; ++j) {
                    const int iv = 2 * j + 1, sv = iv % C::NS, ik = 2 * j + 2, sk = ik % C::NS;
                    const bool more = j + 1 < steps;
                    ok = ptx::mbar_wait(&ctl.full[sv], (iv / C::NS) & 1, abort_flag);
                    if (ok && more)
                        ok = ptx::mbar_wait(&ctl.full[sk], (ik / C::NS) & 1, abort_flag);
                    for (int t = 0; t < tiles && ok; ++t) {
                        const uint64_t vb = smem_desc_mn128(ring + sv * C::STAGE, kTileKeys * 128);
#pragma unroll
                        for (int half = 0; half < 2; ++half) { // (a half of P is multiplied while the other is being formed)
                            ok = ok && ptx::mbar_wait(&ctl.p_full[t][half], j & 1, abort_flag);
                            ptx::tc_fence_after();
                            if (ok)
#pragma unroll
                                for (int k = half * 4; k < half * 4 + 4; ++k)
                                    ptx::mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vb + k * 128, kind_o, j > 0 || k > 0);
                        }
                        if (!ok)
                            break;
                        if (more)
                            scores(t, sk); // over P, whose product is before it in the pipe
                        else
                            ptx::mma_commit(&ctl.o_full[t]);
                    }
                    if (ok) {
                        ptx::mma_commit(&ctl.empty[sv]);
                        if (more)
                            ptx::mma_commit(&ctl.empty[sk]);
                    }
                }
            }
            __syncwarp();
        } else {
            ptx::reg_alloc<kSoftmaxRegs>();
            // ---- softmax: a thread owns row 32 (warp & 3) + lane of its tile ---------------------------------------------------
            const int t = warp >> 2, r = t * kTileRows + (warp & 3) * 32 + lane, tok = (row0 + r) / a.group, hd = row0 + r - tok * a.group;
            if (t < tiles) {
                const bool live = r < rows;
                const int lim = live ? a.s.visible(tok, ql, own, a.causal) - n0 : own_last; // of its own keys (rows past the end: zeros of q, nothing is written)
                const int warp_lim = __reduce_min_sync(0xffffffffu, lim);
                const uint32_t lanes = (uint32_t)(warp & 3) << 21, s_t = tmem + lanes + t * 128, o_t = tmem + lanes + 256 + t * 128;
                float m = -INFINITY, l = 0.f; // m: the maximum in use, times scale log2(e), as lifted() leaves it
                bool ok = true;
                for (int j = 0; j < steps; ++j) {
                    ok = ptx::mbar_wait_warp(&ctl.s_full[t], j & 1, abort_flag);
                    if (!ok)
                        break;
                    ptx::tc_fence_after();
                    uint32_t s[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        ptx::tmem_ld_32x32(s_t + c * 32, s[c]);
                    ptx::tmem_ld_wait();
                    const int jj = k0 + j, key0 = first_key(jj);
                    if (key0 + kTileKeys > (jj < tiles0 ? n0 : warp_lim)) {
                        const int see = (jj < tiles0 ? n0 : lim) - key0;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                s[c][i] = c * 32 + i < see ? s[c][i] : 0xff800000u;
                    }
                    float mx[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
                        for (int i = 1; i < 31; i += 2)
                            mx[c] = ptx::max3_nan(mx[c], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                        mx[c] = ptx::max3_nan(mx[c], mx[c], __uint_as_float(s[c][31]));
                    }
                    float top = ptx::max3_nan(ptx::max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * a.sl2;
                    if (!(top < INFINITY))
                        top = NAN; // the formula's inf - inf, or a score that is none: the row's result is NaN
                    // Below, a score's product with the scale is not rounded, as m is: of a score t the difference is up to 2^-24 t, which would
                    // be a power out of range where t is large.  Such scores are rounded first.
                    float2 sl2 = make_float2(a.sl2, a.sl2);
                    if (__any_sync(0xffffffffu, fabsf(top) >= kLargePower && top > -INFINITY)) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                s[c][i] = __float_as_uint(__uint_as_float(s[c][i]) * a.sl2);
                        sl2 = make_float2(1.f, 1.f);
                    }
                    top = lifted<T>(top, 7.f); // (and up to 2^8 more while the maximum grows: 2^15 of fp16's 2^16)
                    if (j == 0)
                        m = top;
                    else if (__any_sync(0xffffffffu, top - m > kGrowth || top != top)) {
                        // (the product with the tile before is done: its scores' successor was behind it in the pipe)
                        const float to = top != top || m != m ? NAN : fmaxf(m, top), f = m == to ? 1.f : exp2_approx(m - to);
                        m = to;
                        l *= f;
#pragma unroll
                        for (int c = 0; c < DP / 16; ++c) {
                            uint32_t o[16];
                            ptx::tmem_ld_32x16(o_t + c * 16, o);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            ptx::tmem_st_32x16(o_t + c * 16, o);
                        }
                    }
                    const float z = m == -INFINITY ? 0.f : -m;
                    const float2 zz = make_float2(z, z);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float2 x = ptx::fma_f32x2(make_float2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), sl2, zz);
                            x.x = exp2_approx(x.x), x.y = exp2_approx(x.y);
                            sum[i & 1] = ptx::add_f32x2(sum[i & 1], x);
                            p[i] = pack2<T>(x.x, x.y);
                        }
                        ptx::tmem_st_32x16(s_t + c * 16, p);
                        if (c & 1) {
                            ptx::tmem_st_wait();
                            ptx::tc_fence_before();
                            ptx::mbar_arrive(&ctl.p_full[t][c >> 1]);
                        }
                    }
                    sum[0] = ptx::add_f32x2(sum[0], sum[1]);
                    l += sum[0].x + sum[0].y;
                }
                // ---- the rows' results --------------------------------------------------------------------------------------
                if (ok && steps > 0)
                    ok = ptx::mbar_wait_warp(&ctl.o_full[t], 0, abort_flag);
                if (ok) {
                    ptx::tc_fence_after();
                    const int key_a = max(k0 - tiles0, 0) * kTileKeys, key_b = min(lim, (k1 - tiles0) * kTileKeys); // its own keys here
                    const bool seen = steps > 0 && (k0 < tiles0 || key_b > key_a); // this row sees some of this block's keys
                    const long long grow = (long long)(t0 + tok) * a.group + hd, at = ((long long)split * a.hkv + h) * ((long long)a.s.tokens * a.group) + grow;
                    const bool bad = steps > 0 && *(volatile int *)&ctl.bad;
                    const float inv = 1.f / l;
                    if (to_pieces && live)
                        a.pml[at] = make_float2(seen ? fmaxf(m, -FLT_MAX) : -INFINITY, l);
                    T *out = (T *)a.out + (long long)(t0 + tok) * a.o_tok + (long long)(h * a.group + hd) * a.o_head;
#pragma unroll 1
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t o[32];
                        if (steps > 0) {
                            ptx::tmem_ld_32x32(o_t + c * 32, o);
                            ptx::tmem_ld_wait();
                        }
                        if (!seen) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                o[i] = 0u;
                        }
                        if (bad && live) {
                            for (int key = max(key_a, own_first / kTileKeys * kTileKeys); key < key_b; ++key) {
                                int slot;
                                const int p = a.s.page(b, n0 + key, slot);
                                const T *v = (const T *)a.vc + (long long)p * a.vp + (long long)slot * a.vs + (long long)h * a.vh + c * 32;
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float x = p >= 0 && c * 32 + i < a.dim ? to_f32(v[i]) : 0.f;
                                    if (!(fabsf(x) <= FLT_MAX))
                                        o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
                                }
                            }
                        }
                        if (live && to_pieces) {
                            float4 *po = reinterpret_cast<float4 *>(a.po + at * DP + c * 32);
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                po[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                        } else if (live) {
                            const float f = seen ? inv : 0.f;
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (c * 32 + i * 8 < a.dim) {
                                    uint32_t w[4];
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        w[e] = pack2<T>(__uint_as_float(o[8 * i + 2 * e]) * f, __uint_as_float(o[8 * i + 2 * e + 1]) * f);
                                    *reinterpret_cast<uint4 *>(out + c * 32 + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                                }
                        }
                    }
                }
            }
        }
    }
    // ---- teardown -------------------------------------------------------------------------------------------------------------
    if (*abort_flag) { // copies and products that may still be in flight land before the block's memory is released
        const uint64_t t = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t < 200000ull)
            __nanosleep(1000);
        if (threadIdx.x == 0)
            atomicOr(a.s.status, kStatusWait);
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 15)
        ptx::tmem_dealloc(tmem, 512);
}

// The pool as TMA sees it: boxes of up to 128 slots x 64 values of one page and head.  False where the pages do not fit the tiles.
template <typename T> bool page_map(const PagedArgs &a, const void *pool, long long page, long long slot, long long head, CUtensorMap &map) {
    const int size = a.s.page_size;
    EncodeTiledFn enc = encode_fn();
    if (!enc || size < 8 || a.s.pages < 1 || (size < kTileKeys ? kTileKeys % size : size % kTileKeys))
        return false;
    if ((slot == 0 && size > 1) || (head == 0 && a.hkv > 1) || (page == 0 && a.s.pages > 1)) // (an expanded pool)
        return false;
    auto bytes = [](long long stride) { return (cuuint64_t)(stride ? stride * 2 : 16); }; // (of an extent of one)
    const cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)size, (cuuint64_t)a.hkv, (cuuint64_t)a.s.pages}, strides[3] = {bytes(slot), bytes(head), bytes(page)};
    const cuuint32_t box[4] = {64, (cuuint32_t)std::min(size, kTileKeys), 1, 1}, step[4] = {1, 1, 1, 1};
    if (strides[0] >> 40 || strides[1] >> 40 || strides[2] >> 40)
        return false;
    return enc(&map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(pool), dims,
               strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
int tiles_launch(petb200_ctx *ctx, int dtype, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int pieces_out, cudaStream_t s) {
    using C = TileCfg<DP>;
    const bool one = a.s.kv_lens == nullptr, even = one || !a.s.q_starts;
    const long long rows = (long long)a.s.tokens * a.group;
    const long long tiles = even ? (one ? 1ll : a.s.seqs) * (((long long)(one ? a.s.tokens : a.s.q_len) * a.group + 2 * kTileRows - 1) / (2 * kTileRows))
                                 : rows / (2 * kTileRows) + a.s.seqs;
    const long long units = tiles * a.hkv, keys = (long long)a.s.n0 + (one ? 0 : (long long)a.s.width * a.s.page_size);
    if (keys > 0x7fff0000ll || units > 0x7fff0000ll || rows > 0x7fff0000ll)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "attention over pages: %lld row tiles of up to %lld keys are more than one call takes", units, keys);
    const int splits = pieces_out ? pieces_out : paged_tiles_pieces(ctx, a);
    size_t bytes = 0;
    if (!pieces_out && splits > 1) {
        const size_t po = ((size_t)splits * a.hkv * rows * DP * 4 + 255) & ~(size_t)255;
        a.po = reinterpret_cast<float *>(ws), a.pml = reinterpret_cast<float2 *>(ws + po);
        bytes = po + (size_t)splits * a.hkv * rows * 8;
        a.pieces = splits;
    }
    *need = bytes;
    if (!a.q)
        return PETB200_OK;
    if (bytes > ws_bytes)
        return fail(ctx, PETB200_ERR_INVALID, "attention over pages: a workspace of %zu bytes, %zu are needed", ws_bytes, bytes);
    if (units == 0)
        return PETB200_OK;
    if (int rc = raise_smem(ctx, (const void *)k_paged_tiles<T, DP>, C::SMEM))
        return rc;
    CUtensorMap kmap{}, vmap{};
    const int tma = page_map<T>(a, a.kc, a.kp, a.ks, a.kh, kmap) && page_map<T>(a, a.vc, a.vp, a.vs, a.vh, vmap);
    launch_pdl(k_paged_tiles<T, DP>, dim3((unsigned)(units * splits)), kTileThreads, C::SMEM, s, kmap, vmap, a, splits, (int)(pieces_out || splits > 1), tma, ctx->paged_starve);
    int rc = launched(ctx, "k_paged_tiles");
    if (rc || pieces_out || splits == 1)
        return rc;
    return paged_join_rows(ctx, dtype, a, s);
}

} // namespace

int paged_tiles_wait_limit(unsigned long long ns) {
    return cudaMemcpyToSymbol(ptx::g_mbar_wait_limit_ns, &ns, sizeof ns) == cudaSuccess ? PETB200_OK : PETB200_ERR_CUDA;
}

int paged_tiles_pieces(petb200_ctx *ctx, const PagedArgs &a) {
    const bool one = a.s.kv_lens == nullptr;
    const long long rows = (long long)a.s.tokens * a.group, seqs = one ? 1 : a.s.seqs;
    const long long units = std::max(seqs, (rows + kTileRows) / (2 * kTileRows)) * a.hkv; // about: uneven sequences make a few more
    const long long keys = (long long)a.s.n0 + (one ? 0 : (long long)a.s.width * a.s.page_size);
    // Keys are split until every SM has a block, but no finer than four tiles of them: a piece costs its rows' sums through memory twice.
    return (int)std::max(1ll, std::min({(long long)ctx->sm_count / units, keys / (4 * kTileKeys), 32ll}));
}

int paged_tiles_run(petb200_ctx *ctx, int dtype, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int pieces_out, cudaStream_t s) {
    const bool wide = a.dim > 64;
    if (dtype == PETB200_F16)
        return wide ? tiles_launch<__half, 128>(ctx, dtype, a, ws, ws_bytes, need, pieces_out, s) : tiles_launch<__half, 64>(ctx, dtype, a, ws, ws_bytes, need, pieces_out, s);
    return wide ? tiles_launch<__nv_bfloat16, 128>(ctx, dtype, a, ws, ws_bytes, need, pieces_out, s)
                : tiles_launch<__nv_bfloat16, 64>(ctx, dtype, a, ws, ws_bytes, need, pieces_out, s);
}

} // namespace petb200

// Test hook for the give-up path of k_paged_tiles (not part of the public header; petb200_debug_set_wait_limit shortens the wait): while on, the
// stages of its ring expect one arrival more than there are, so the products' wait runs out, every role leaves and the status word says so.
extern "C" int petb200_debug_paged_starve(petb200_ctx *ctx, int on) {
    if (!ctx)
        return PETB200_ERR_INVALID;
    ctx->paged_starve = on != 0;
    return PETB200_OK;
}
