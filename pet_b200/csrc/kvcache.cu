// A paged cache of keys and values: appending to it, and the checks and choices in front of the attentions that read it.
//
// k_kv_append: out = x turned by its position, pair (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin), and copied to its place.  One pass
// over the data; bound by HBM for prompts, by latency for single tokens.  The angle of a pair is the same for every
// head, so a block first forms the cosines and sines of its tokens in shared memory and then walks the heads in 16-byte pieces.
// Angles: position * frequency in 64 bits, whole turns taken off there (an fp32 product at position 10^5 is off by
// 4 * 10^-3 radians), sincospif of what is left.  The rotation itself is fp32, rounded once to the cache's type.
#include "paged.cuh"
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdlib>

namespace petb200 {
namespace {

constexpr int kAppendThreads = 256, kAppendTokens = 4;

struct AppendArgs {
    PagedSeqs s;
    const void *x[3];                // queries, keys, values
    void *y[3];                      // where they go: q_out, and the two pools
    long long x_tok[3], x_head[3];   // strides in elements
    long long y_tok, y_head[3];      // q_out: token and head; pools: head
    long long y_page[3], y_slot[3];
    int heads[3], dim, rot, interleaved, pos0, tokens_per_block, vec;
    const float *inv_freq;
};

// Eight values as floats; `vec`: the rows are on the 16-byte grid.
template <typename S> __device__ __forceinline__ void load8(const S *p, bool vec, float (&v)[8]) {
    if (vec) {
        uint4 w[sizeof(S) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(S) / 2; ++i)
            w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        const S *e = reinterpret_cast<const S *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = to_f32(p[i]);
    }
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    uint4 w[sizeof(T) / 2];
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4 *>(p)[i] = w[i];
}

template <typename S, typename T> __global__ void __launch_bounds__(kAppendThreads) k_kv_append(const AppendArgs a) {
    pdl_prologue();
    __shared__ float2 turn[kAppendTokens][kPagedMaxDim / 2]; // {cos, sin}
    __shared__ int where[kAppendTokens][3];                  // page (-1: nowhere), slot, whether the row belongs to a sequence
    __shared__ int position[kAppendTokens];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tok0 = blockIdx.x * a.tokens_per_block, ntok = min(a.tokens_per_block, a.s.tokens - tok0);
    if (warp < ntok) {
        const int t = tok0 + warp;
        int b;
        if (a.s.q_starts) { // the last sequence that begins at or before t: as many as do, up to 1024 of them looked at together
            int from = 0, most = a.s.seqs + 1, n = 0;
            while (most > 1024) { // (32 probes narrow down where more are)
                const int step = ceil_div(most, 32), i = from + lane * step;
                const int c = __popc(__ballot_sync(0xffffffffu, lane * step < most && __ldg(a.s.q_starts + i) <= t));
                const int skip = max(c - 1, 0) * step;
                from += skip, most = min(step, most - skip);
            }
            for (int i = lane; i < most; i += 32)
                n += __ldg(a.s.q_starts + from + i) <= t;
            b = from + (int)__reduce_add_sync(0xffffffffu, n) - 1;
        } else
            b = t / a.s.q_len;
        if (lane == 0) {
            int page = -1, slot = 0, in = 0, p = 0, t0 = 0;
            if (b >= 0 && b < a.s.seqs) {
                const int n = a.s.span(b, t0);
                if (t >= t0 && t < t0 + n) {
                    in = 1;
                    p = __ldg(a.s.kv_lens + b) - n + (t - t0);
                    if (p >= 0 && a.s.page_of(p) < a.s.width)
                        page = a.s.page(b, p, slot);
                    else if (p >= 0)
                        atomicOr(a.s.status, kStatusPage);
                }
            }
            where[warp][0] = page, where[warp][1] = slot, where[warp][2] = in;
            position[warp] = p;
        }
    }
    __syncthreads();
    const int half = a.rot / 2;
    for (int i = threadIdx.x; i < ntok * half; i += kAppendThreads) {
        const int t = i / half, j = i - t * half;
        const double turns = ((double)a.pos0 + (double)position[t]) * (double)__ldg(a.inv_freq + j) * 0.15915494309189533577; // 1 / (2 pi)
        float sn, cs;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
        turn[t][j] = make_float2(cs, sn);
    }
    __syncthreads();
    // A thread takes two 16-byte pieces of a head at a time, so that the halves of a pair are read once: pieces d and d + half where
    // that is how values pair up, neighbours elsewhere (values, interleaved pairs, what is not turned).  Eight threads or fewer share
    // a head of 128; `step` (token, head) pairs are walked at once, two rounds of loads ahead of their stores.
    const int per_head = (a.dim + 15) / 16, group = threadIdx.x / per_head, step = kAppendThreads / per_head, e = threadIdx.x - group * per_head;
    const int heads = a.heads[0] + a.heads[1] + a.heads[2], turned = a.interleaved || (half & 7) ? 0 : half / 8; // piece pairs that are halves
    if (group >= step)
        return;
    struct Two {
        float v[2][8];
        const S *x; // the head's values
        T *y;       // where they go; null: nowhere
        int d[2], t, kind;
    };
    auto fetch = [&](int i, Two &w) {
        const int t = i / heads, hh = i - t * heads;
        w.y = nullptr;
        if (t >= ntok)
            return;
        w.kind = hh < a.heads[0] ? 0 : hh < a.heads[0] + a.heads[1] ? 1 : 2, w.t = t;
        const int h = hh - (w.kind > 0 ? a.heads[0] : 0) - (w.kind > 1 ? a.heads[1] : 0), page = where[t][0];
        if (w.kind ? page < 0 : !where[t][2])
            return;
        if (w.kind < 2 && turned)
            w.d[0] = e < turned ? e * 8 : a.rot + (e - turned) * 16, w.d[1] = w.d[0] + (e < turned ? half : 8);
        else
            w.d[0] = e * 16, w.d[1] = e * 16 + 8;
        w.x = (const S *)a.x[w.kind] + (long long)(tok0 + t) * a.x_tok[w.kind] + (long long)h * a.x_head[w.kind];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (w.d[k] < a.dim)
                load8(w.x + w.d[k], a.vec, w.v[k]);
        w.y = (T *)a.y[w.kind] + (long long)h * a.y_head[w.kind] +
              (w.kind ? (long long)page * a.y_page[w.kind] + (long long)where[t][1] * a.y_slot[w.kind] : (long long)(tok0 + t) * a.y_tok);
    };
    auto put = [&](Two &w) {
        if (!w.y)
            return;
        if (w.kind < 2) {
            const float2 *c = turn[w.t];
            if (turned) {
                if (e < turned)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 cs = c[e * 8 + k];
                        const float x1 = w.v[0][k], x2 = w.v[1][k];
                        w.v[0][k] = x1 * cs.x - x2 * cs.y, w.v[1][k] = x2 * cs.x + x1 * cs.y;
                    }
            } else if (a.interleaved) {
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int k = 0; k < 8; k += 2)
                        if (w.d[p] + k < a.rot) {
                            const float2 cs = c[(w.d[p] + k) >> 1];
                            const float x1 = w.v[p][k], x2 = w.v[p][k + 1];
                            w.v[p][k] = x1 * cs.x - x2 * cs.y, w.v[p][k + 1] = x2 * cs.x + x1 * cs.y;
                        }
            } else { // halves that do not fall on pieces: the other value of each pair is read by itself
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int d = w.d[p] + k;
                        if (d < a.rot) {
                            const bool low = d < half;
                            const float2 cs = c[low ? d : d - half];
                            const float o = to_f32(w.x[low ? d + half : d - half]);
                            w.v[p][k] = low ? w.v[p][k] * cs.x - o * cs.y : w.v[p][k] * cs.x + o * cs.y;
                        }
                    }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (w.d[k] < a.dim)
                store8(w.y + w.d[k], w.v[k]);
    };
    const int all = ntok * heads;
    for (int i = blockIdx.y * step + group; i < all; i += 2 * gridDim.y * step) {
        Two p, q;
        fetch(i, p);
        fetch(i + gridDim.y * step, q);
        put(p);
        put(q);
    }
}

template <typename S, typename T> int append_launch(petb200_ctx *ctx, AppendArgs &a, cudaStream_t s) {
    const int heads = a.heads[0] + a.heads[1] + a.heads[2], step = kAppendThreads / ((a.dim + 15) / 16);
    // Several tokens to a block share its angles and barriers; few tokens are spread over blocks instead, a head or two a thread.
    a.tokens_per_block = a.s.tokens >= kAppendTokens * 2 * ctx->sm_count ? kAppendTokens : 1;
    const int blocks = ceil_div(a.s.tokens, a.tokens_per_block);
    const int split = blocks < 4 * ctx->sm_count ? std::min(ceil_div(heads, step), 64) : 1;
    launch_pdl(k_kv_append<S, T>, dim3((unsigned)blocks, (unsigned)split), kAppendThreads, 0, s, a);
    return launched(ctx, "k_kv_append");
}

int type_size(int dtype) { return dtype == PETB200_F32 ? 4 : 2; }
bool on_grid(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Restores the calling thread's device: a call is made on the context's, whichever is current.
struct DeviceGuard {
    int was = -1;
    bool moved = false;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&was) == cudaSuccess && was != device)
            moved = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceGuard() {
        if (moved)
            (void)cudaSetDevice(was);
    }
};

// The stride of an extent of one is never used, and may be anything.
petb200_kv_cache plain_strides(petb200_kv_cache c) {
    if (c.pages <= 1)
        c.k_page = c.v_page = 0;
    if (c.page_size == 1)
        c.k_slot = c.v_slot = 0;
    if (c.heads == 1)
        c.k_head = c.v_head = 0;
    return c;
}
petb200_kv_rows plain_strides(const petb200_kv_rows *rows, int tokens, int heads) {
    petb200_kv_rows r = rows ? *rows : petb200_kv_rows{};
    if (tokens <= 1)
        r.tok = 0;
    if (heads <= 1)
        r.head = 0;
    return r;
}

// Whether two sets of rows [tokens, heads, dim] have a byte in common; `bytes` of a row, strides in bytes.  Rows of one merged tensor, side by
// side in every token, have not, although their ranges meet.  (Ranges that meet with different token strides count as overlapping.)
struct ByteRows {
    uintptr_t p;
    long long tok, head, bytes;
    int heads;
};
bool rows_overlap(ByteRows a, ByteRows b, int tokens) {
    long long lo[2], hi[2], head_lo[2], head_hi[2]; // of all rows, and of one token's, from a.p
    const ByteRows *r[2] = {&a, &b};
    const long long apart = (long long)(b.p - a.p);
    for (int i = 0; i < 2; ++i) {
        const long long t = r[i]->tok * (tokens - 1), h = r[i]->head * (r[i]->heads - 1), at = i ? apart : 0;
        head_lo[i] = at + std::min(h, 0ll), head_hi[i] = at + std::max(h, 0ll) + r[i]->bytes;
        lo[i] = head_lo[i] + std::min(t, 0ll), hi[i] = head_hi[i] + std::max(t, 0ll);
    }
    if (lo[0] >= hi[1] || lo[1] >= hi[0])
        return false;
    if (a.tok != b.tok)
        return true;
    // Whether some token of b, k strides on, reaches into [x, x + n) from [y, y + m).
    const long long step = std::abs(a.tok);
    auto meet = [&](long long x, long long n, long long y, long long m) {
        if (step == 0)
            return y < x + n && x < y + m;
        const long long d = x - m - y; // the first k with y + k step > x - m
        const long long k = d >= 0 ? d / step + 1 : -((-d - 1) / step);
        return std::max(k, 1ll - tokens) <= tokens - 1 && y + std::max(k, 1ll - tokens) * step < x + n;
    };
    if (!meet(head_lo[0], head_hi[0] - head_lo[0], head_lo[1], head_hi[1] - head_lo[1]))
        return false;
    for (int i = 0; i < a.heads; ++i)
        for (int j = 0; j < b.heads; ++j)
            if (meet(i * a.head, a.bytes, apart + j * b.head, b.bytes))
                return true;
    return false;
}
bool rows_overlap(const petb200_kv_rows &a, int a_heads, int a_dtype, const petb200_kv_rows &b, int b_heads, int b_dtype, int dim, int tokens) {
    const long long sa = type_size(a_dtype), sb = type_size(b_dtype);
    return rows_overlap({(uintptr_t)a.p, a.tok * sa, a.head * sa, dim * sa, a_heads}, {(uintptr_t)b.p, b.tok * sb, b.head * sb, dim * sb, b_heads}, tokens);
}

int check_cache(petb200_ctx *ctx, const char *what, const petb200_kv_cache *cache, const petb200_kv_seqs *s) {
    if (!cache || !s)
        return fail(ctx, PETB200_ERR_INVALID, "%s: null argument", what);
    const petb200_kv_cache plain = plain_strides(*cache), *c = &plain;
    if (c->dtype < PETB200_F32 || c->dtype > PETB200_BF16)
        return fail(ctx, PETB200_ERR_INVALID, "%s: unknown type %d", what, c->dtype);
    if (c->pages < 0 || c->page_size <= 0 || c->heads <= 0 || c->dim <= 0 || s->seqs < 0 || s->tokens < 0 || s->table_width < 0)
        return fail(ctx, PETB200_ERR_INVALID, "%s: a size is negative or zero", what);
    if (c->dim % 8 || c->dim > kPagedMaxDim)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: head widths are multiples of 8 up to %d (got %d)", what, kPagedMaxDim, c->dim);
    const long long e = 16 / type_size(c->dtype);
    if (!on_grid(c->k) || !on_grid(c->v) || c->k_page % e || c->k_slot % e || c->k_head % e || c->v_page % e || c->v_slot % e || c->v_head % e)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: the pools and their strides must be multiples of 16 bytes", what);
    if (c->k_page < 0 || c->k_slot < 0 || c->k_head < 0 || c->v_page < 0 || c->v_slot < 0 || c->v_head < 0 || s->table_stride < 0)
        return fail(ctx, PETB200_ERR_INVALID, "%s: negative strides", what);
    if ((long long)s->table_width * c->page_size > 0x7fff0000ll)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: a table row of %d pages of %d keys: more than 2^31 keys", what, s->table_width, c->page_size);
    if (s->seqs && s->tokens) {
        if ((s->table_width && !s->page_table) || !s->kv_lens)
            return fail(ctx, PETB200_ERR_INVALID, "%s: no page table or no lengths", what);
        if (!c->pages || !c->k || !c->v)
            return fail(ctx, PETB200_ERR_INVALID, "%s: a cache without pages", what);
        if (!s->q_starts && s->tokens % s->seqs)
            return fail(ctx, PETB200_ERR_INVALID, "%s: %d tokens are not the same number for each of %d sequences", what, s->tokens, s->seqs);
    }
    return PETB200_OK;
}

PagedSeqs device_seqs(petb200_ctx *ctx, const petb200_kv_cache *c, const petb200_kv_seqs *s) {
    PagedSeqs d;
    d.table = s->page_table, d.tstride = s->table_stride, d.width = s->table_width;
    d.kv_lens = s->kv_lens, d.q_starts = s->q_starts, d.seqs = s->seqs, d.tokens = s->tokens;
    d.q_len = s->seqs ? s->tokens / s->seqs : 0;
    d.page_size = c->page_size, d.pages = c->pages, d.status = ctx->d_status;
    d.page_shift = -1;
    if ((c->page_size & (c->page_size - 1)) == 0)
        for (d.page_shift = 0; (1 << d.page_shift) < c->page_size;)
            ++d.page_shift;
    return d;
}

PagedArgs attention_args(petb200_ctx *ctx, const petb200_kv_cache *cache, const petb200_kv_seqs *s, int q_heads) {
    PagedArgs a;
    const petb200_kv_cache plain = plain_strides(*cache), *c = &plain;
    a.s = device_seqs(ctx, c, s);
    a.kc = c->k, a.vc = c->v;
    a.kp = c->k_page, a.ks = c->k_slot, a.kh = c->k_head, a.vp = c->v_page, a.vs = c->v_slot, a.vh = c->v_head;
    a.hkv = c->heads, a.group = q_heads / c->heads, a.dim = c->dim;
    return a;
}

// Rows of a sequence and key head from which a 128-row tile is used, be it part full: as soon as 16 rows are not enough, and its keys would
// be read again.  16 sequences of 4000 keys, 8 key heads of 128, us with 16-row tiles / 128-row tiles: 16 rows 57 / 66, 32 rows 85 / 67,
// 64 rows 147 / 68; 32 sequences of 700 keys: 33 / 36, 49 / 36, 67 / 36.
constexpr int kTileFrom = 17;
// Rows from which a sequence behind a shared prefix reads it by itself: a row for every 48 shared keys, at most 192.  Rows that go together
// fill their tiles but meet their own keys in 16-row tiles; alone a sequence's tile is part empty for all of the prefix.  fp16, us
// together / alone, width 128: 16 sequences behind 4000 keys, 20 own beside the new ones: 48 rows 57 / 74, 96 rows 66 / 74, 128 rows 84 / 74; 16
// behind 8200: 128 rows 117 / 135, 168 rows 184 / 146; 8 behind 16000: 168 rows 129 / 148, 192 rows 131 / 148, 240 rows 176 / 150; 32 behind
// 1000: 24 rows 57 / 51.  Width 64: 16 behind 4000: 48 rows 41 / 39, 128 rows 57 / 39; 16 behind 8200: 96 rows 55 / 61, 128 rows 70 / 61, 168
// rows 70 / 72, 192 rows 72 / 74, 240 rows 94 / 74; 8 behind 16000: 128 rows 57 / 59, 168 rows 92 / 70.  What goes together moves in steps, as
// the tiles of all rows fill the GPU once or twice, so no one border is right everywhere: near it the rule loses up to a quarter.
long long alone_from(int prefix_len) { return std::min(192, std::max(kTileFrom, prefix_len / 48)); }

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Attention over the sequences' own keys behind `prefix_len` shared ones, or (a.q == nullptr) the workspace that it takes.
int attend(petb200_ctx *ctx, int dtype, PagedArgs a, const int *prefix_table, int prefix_len, char *ws, size_t ws_bytes, size_t *need, cudaStream_t s) {
    const long long rows = (long long)a.s.tokens * a.group;
    a.s.table0 = prefix_table;
    a.s.n0 = prefix_len;
    const bool halves = dtype != PETB200_F32;
    const long long each = rows / a.s.seqs;
    // A sequence with rows enough for tiles of its own gains nothing from the others: its keys, shared and own, are read as one run.
    if (prefix_len == 0 || a.s.seqs == 1 || each >= alone_from(prefix_len))
        return halves && each >= kTileFrom ? paged_tiles_run(ctx, dtype, a, ws, ws_bytes, need, 0, s) : paged_rows_run(ctx, dtype, a, ws, ws_bytes, need, 0, s);
    // All tokens as one sequence against the shared keys, in pieces; each sequence against its own, as one more piece; the pieces of a row added.
    PagedArgs p = a;
    p.s.kv_lens = nullptr, p.s.q_starts = nullptr;
    // (16-row tiles share their launch with the own keys, and are done before a second launch: 32 rows against 1901 keys 16 us, 26 in tiles)
    const bool tiles = halves && rows >= 64;
    int pieces;
    if (tiles)
        pieces = paged_tiles_pieces(ctx, p);
    else {
        const long long units = (rows + 15) / 16 * a.hkv;
        pieces = (int)std::max(1ll, std::min({(2ll * ctx->sm_count + units - 1) / units, (prefix_len + 255ll) / 256, 64ll}));
    }
    const int dp = a.dim > 64 ? 128 : 64;
    const size_t po = align256((size_t)(pieces + 1) * a.hkv * rows * dp * 4), pml = align256((size_t)(pieces + 1) * a.hkv * rows * 8);
    p.po = a.po = reinterpret_cast<float *>(ws);
    p.pml = a.pml = reinterpret_cast<float2 *>(ws + po);
    a.pieces = pieces + 1, a.piece_out = pieces;
    size_t more = 0;
    const bool ask = !a.q;
    if (!ask && po + pml > ws_bytes)
        return fail(ctx, PETB200_ERR_INVALID, "attention over pages: a workspace of %zu bytes is too small", ws_bytes);
    if (tiles) {
        if (int rc = paged_tiles_run(ctx, dtype, p, nullptr, 0, &more, pieces, s))
            return rc;
        a.s.n0 = 0;
    }
    int rc = paged_rows_run(ctx, dtype, a, ask ? nullptr : ws + po + pml, ask ? 0 : ws_bytes - po - pml, &more, tiles ? 0 : pieces, s);
    *need = po + pml + more;
    return rc || ask ? rc : paged_join_rows(ctx, dtype, a, s);
}

int attention_run(petb200_ctx *ctx, const char *what, const petb200_kv_cache *cache, const petb200_kv_seqs *seqs, const int *prefix_table,
                  int prefix_len, const petb200_kv_rows *q_rows, const petb200_kv_rows *out_rows, int q_heads, int causal, float scale, void *workspace,
                  size_t workspace_bytes, cudaStream_t s) {
    if (!ctx)
        return PETB200_ERR_INVALID;
    if (int rc = check_cache(ctx, what, cache, seqs))
        return rc;
    if (q_heads <= 0 || q_heads % cache->heads)
        return fail(ctx, PETB200_ERR_INVALID, "%s: %d query heads on %d key heads", what, q_heads, cache->heads);
    const float sl2 = scale * 1.44269504088896340736f; // log2(e)
    if (!std::isfinite(sl2) || scale < FLT_MIN)
        return fail(ctx, PETB200_ERR_INVALID, "%s: the scale must be positive, finite (its product with log2(e) too) and not denormal", what);
    if (seqs->seqs == 0 || seqs->tokens == 0)
        return PETB200_OK;
    const petb200_kv_rows q = plain_strides(q_rows, seqs->tokens, q_heads), out = plain_strides(out_rows, seqs->tokens, q_heads);
    if (!q.p || !out.p || (prefix_len > 0 && !prefix_table))
        return fail(ctx, PETB200_ERR_INVALID, "%s: null argument", what);
    const long long e = 16 / type_size(cache->dtype);
    if (!on_grid(q.p) || !on_grid(out.p) || q.tok % e || q.head % e || out.tok % e || out.head % e || q.tok < 0 || q.head < 0 || out.tok < 0 || out.head < 0)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: rows of q and out must start on 16-byte boundaries", what);
    if (rows_overlap(q, q_heads, cache->dtype, out, q_heads, cache->dtype, cache->dim, seqs->tokens))
        return fail(ctx, PETB200_ERR_INVALID, "%s: out must not overlap q", what);
    if (!on_grid(workspace))
        return fail(ctx, PETB200_ERR_INVALID, "%s: the workspace must be 16-byte aligned", what);
    DeviceGuard guard(ctx->device);
    PagedArgs a = attention_args(ctx, cache, seqs, q_heads);
    a.q = q.p, a.q_tok = q.tok, a.q_head = q.head;
    a.out = out.p, a.o_tok = out.tok, a.o_head = out.head;
    a.causal = causal != 0;
    a.sl2 = sl2;
    size_t need = 0;
    return attend(ctx, cache->dtype, a, prefix_table, prefix_len, (char *)workspace, workspace ? workspace_bytes : 0, &need, s);
}

} // namespace
} // namespace petb200

using namespace petb200;

extern "C" int petb200_kv_append_run(petb200_ctx *ctx, const petb200_kv_cache *cache, const petb200_kv_seqs *seqs, const petb200_kv_rows *k,
                                     const petb200_kv_rows *v, const petb200_kv_rows *q, const petb200_kv_rows *q_out, int q_heads, int src_dtype,
                                     const float *inv_freq, int rotary, int interleaved, int pos0, petb200_stream stream) {
    const char *what = "kv_append";
    if (!ctx)
        return PETB200_ERR_INVALID;
    if (int rc = check_cache(ctx, what, cache, seqs))
        return rc;
    if (src_dtype != cache->dtype && src_dtype != PETB200_F32)
        return fail(ctx, PETB200_ERR_INVALID, "%s: sources are of the cache's type or fp32", what);
    if (!inv_freq)
        rotary = 0;
    if (rotary < 0 || rotary > cache->dim || rotary % 2)
        return fail(ctx, PETB200_ERR_INVALID, "%s: %d values of %d cannot be turned in pairs", what, rotary, cache->dim);
    const int tokens = seqs->tokens;
    const petb200_kv_rows src[3] = {plain_strides(q, tokens, q_heads), plain_strides(k, tokens, cache->heads), plain_strides(v, tokens, cache->heads)};
    const petb200_kv_rows to = plain_strides(q_out, tokens, q_heads);
    const bool with_q = src[0].p != nullptr;
    if (q_heads < 0 || (with_q && q_heads == 0))
        return fail(ctx, PETB200_ERR_INVALID, "%s: %d query heads", what, q_heads);
    if (seqs->seqs == 0 || seqs->tokens == 0)
        return PETB200_OK;
    if (!src[1].p || !src[2].p || (with_q && !to.p))
        return fail(ctx, PETB200_ERR_INVALID, "%s: null argument", what);
    const long long e = 16 / type_size(cache->dtype), es = 16 / type_size(src_dtype);
    if (with_q && (!on_grid(to.p) || to.tok % e || to.head % e || to.tok < 0 || to.head < 0))
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: rows of q_out must start on 16-byte boundaries", what);
    for (int i = 0; with_q && i < 3; ++i)
        if (rows_overlap(src[i], i ? cache->heads : q_heads, src_dtype, to, q_heads, cache->dtype, cache->dim, tokens))
            return fail(ctx, PETB200_ERR_INVALID, "%s: q_out must not overlap a source", what);
    AppendArgs a{};
    a.s = device_seqs(ctx, cache, seqs);
    a.vec = 1;
    for (int i = 0; i < 3; ++i) {
        a.heads[i] = i ? cache->heads : (with_q ? q_heads : 0);
        a.x[i] = src[i].p, a.x_tok[i] = src[i].tok, a.x_head[i] = src[i].head;
        if (a.heads[i] && (!on_grid(src[i].p) || src[i].tok % es || src[i].head % es))
            a.vec = 0;
    }
    a.y[0] = to.p, a.y_tok = to.tok, a.y_head[0] = to.head;
    const petb200_kv_cache c = plain_strides(*cache);
    a.y[1] = c.k, a.y_page[1] = c.k_page, a.y_slot[1] = c.k_slot, a.y_head[1] = c.k_head;
    a.y[2] = c.v, a.y_page[2] = c.v_page, a.y_slot[2] = c.v_slot, a.y_head[2] = c.v_head;
    a.dim = cache->dim, a.rot = rotary, a.interleaved = interleaved != 0, a.pos0 = pos0, a.inv_freq = inv_freq;
    if ((long long)(a.heads[0] + a.heads[1] + a.heads[2]) * a.dim > 1 << 24)
        return fail(ctx, PETB200_ERR_UNSUPPORTED, "%s: a token of more than 2^24 values", what);
    DeviceGuard guard(ctx->device);
    const cudaStream_t s = (cudaStream_t)stream;
    if (cache->dtype == PETB200_F32)
        return append_launch<float, float>(ctx, a, s);
    if (cache->dtype == PETB200_F16)
        return src_dtype == PETB200_F32 ? append_launch<float, __half>(ctx, a, s) : append_launch<__half, __half>(ctx, a, s);
    return src_dtype == PETB200_F32 ? append_launch<float, __nv_bfloat16>(ctx, a, s) : append_launch<__nv_bfloat16, __nv_bfloat16>(ctx, a, s);
}

extern "C" int petb200_attention_paged_run(petb200_ctx *ctx, const petb200_kv_cache *cache, const petb200_kv_seqs *seqs, const petb200_kv_rows *q,
                                           const petb200_kv_rows *out, int q_heads, int causal, float scale, void *workspace,
                                           size_t workspace_bytes, petb200_stream stream) {
    return attention_run(ctx, "attention_paged", cache, seqs, nullptr, 0, q, out, q_heads, causal, scale, workspace, workspace_bytes,
                         (cudaStream_t)stream);
}

extern "C" int petb200_attention_prefix_run(petb200_ctx *ctx, const petb200_kv_cache *cache, const petb200_kv_seqs *seqs,
                                            const int *prefix_table, int prefix_len, const petb200_kv_rows *q, const petb200_kv_rows *out, int q_heads,
                                            int causal, float scale, void *workspace, size_t workspace_bytes, petb200_stream stream) {
    if (ctx && prefix_len < 0)
        return fail(ctx, PETB200_ERR_INVALID, "attention_prefix: a prefix of %d keys", prefix_len);
    return attention_run(ctx, "attention_prefix", cache, seqs, prefix_table, prefix_len, q, out, q_heads, causal, scale, workspace,
                         workspace_bytes, (cudaStream_t)stream);
}

extern "C" int petb200_attention_paged_workspace(petb200_ctx *ctx, const petb200_kv_cache *cache, const petb200_kv_seqs *seqs, int prefix_len,
                                                 int q_heads, size_t *bytes) {
    if (!ctx)
        return PETB200_ERR_INVALID;
    if (!bytes || prefix_len < 0)
        return fail(ctx, PETB200_ERR_INVALID, "attention_paged_workspace: bad arguments");
    *bytes = 0;
    if (int rc = check_cache(ctx, "attention_paged_workspace", cache, seqs))
        return rc;
    if (q_heads <= 0 || q_heads % cache->heads)
        return fail(ctx, PETB200_ERR_INVALID, "attention_paged_workspace: %d query heads on %d key heads", q_heads, cache->heads);
    if (seqs->seqs == 0 || seqs->tokens == 0)
        return PETB200_OK;
    return attend(ctx, cache->dtype, attention_args(ctx, cache, seqs, q_heads), nullptr, prefix_len, nullptr, 0, bytes, nullptr);
}

// Test hook (not part of the public header): the check of outputs against inputs, on numbers alone.  rows: {address, token stride, head stride,
// heads, bytes of a row} of either, in bytes.
extern "C" int petb200_debug_rows_overlap(const long long *a, const long long *b, int tokens) {
    auto rows = [](const long long *r) { return ByteRows{(uintptr_t)r[0], r[1], r[2], r[4], (int)r[3]}; };
    return rows_overlap(rows(a), rows(b), tokens);
}
