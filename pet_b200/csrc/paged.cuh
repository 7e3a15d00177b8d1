// What the kernels over a paged cache of keys and values share: how a token finds its sequence, a sequence its keys and a key
// its page (kvcache.cu appends, paged_rows.cu and paged_tiles.cu attend).
#pragma once
#include "common.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace petb200 {

constexpr int kPagedMaxDim = 128; // head widths served: multiples of 8 up to this (a row is whole 16-byte pieces)

// Sequences of one call.  Lengths and tables live on the device; the host knows only how much there can be.
struct PagedSeqs {
    const int *table = nullptr, *table0 = nullptr; // pages of each sequence's own keys; of the keys that all of them begin with
    long long tstride = 0;
    const int *kv_lens = nullptr, *q_starts = nullptr;
    int width = 0, n0 = 0, q_len = 0, seqs = 0, tokens = 0;
    int page_size = 1, page_shift = -1, pages = 0;
    int *status = nullptr;

    // Tokens [t0, t0 + n) of sequence b.  Starts that run backwards or past the tokens give fewer tokens, never others' memory.
    __device__ __forceinline__ int span(int b, int &t0) const {
        if (!q_starts) {
            t0 = b * q_len;
            return q_len;
        }
        t0 = min(max(__ldg(q_starts + b), 0), tokens);
        return min(max(__ldg(q_starts + b + 1), t0), tokens) - t0;
    }
    // Keys of its own that sequence b has.
    __device__ __forceinline__ int own(int b) const {
        if (!kv_lens)
            return 0;
        const int n = __ldg(kv_lens + b), most = width * page_size;
        if (n > most)
            atomicOr(status, kStatusPage);
        return min(max(n, 0), most);
    }
    __device__ __forceinline__ int page_of(int key) const { return page_shift >= 0 ? key >> page_shift : key / page_size; }
    // The table's entry for key `key` of sequence b (keys [0, n0) are the shared ones), the key's place in that page in `slot`.
    __device__ __forceinline__ int entry(int b, int key, int &slot) const {
        const int own_key = key - n0;
        const int k = own_key < 0 ? key : own_key, i = page_of(k);
        slot = k - i * page_size;
        return own_key < 0 ? __ldg(table0 + i) : __ldg(table + b * tstride + i);
    }
    __device__ __forceinline__ bool is_page(int p) const { return (unsigned)p < (unsigned)pages; }
    // The page, or -1 (reported) where the entry is none.
    __device__ __forceinline__ int page(int b, int key, int &slot) const {
        const int p = entry(b, key, slot);
        if (is_page(p))
            return p;
        atomicOr(status, kStatusPage);
        return -1;
    }
    // Keys that token i of n sees, of n0 + own: all shared ones, and its own up to the one that came with it.
    __device__ __forceinline__ int visible(int i, int n, int own, int causal) const {
        return n0 + (causal ? min(max(own - n + i + 1, 0), own) : own);
    }
};

struct PagedArgs {
    PagedSeqs s;
    const void *q = nullptr, *kc = nullptr, *vc = nullptr;
    void *out = nullptr;
    long long q_tok = 0, q_head = 0, o_tok = 0, o_head = 0; // strides in elements
    long long kp = 0, ks = 0, kh = 0, vp = 0, vs = 0, vh = 0; // of the cache: page, slot, head
    int hkv = 0, group = 1, dim = 0, causal = 0;
    float sl2 = 0.f; // scale * log2(e): the softmax runs on powers of two
    // Pieces: a row's sum over part of its keys, O unnormalised [piece][hkv][rows][DP] with {m, l} beside it, rows = tokens * group.
    // m is the largest score * sl2 (less the offset of lifted()); -inf: the row sees none of these keys, -FLT_MAX: it sees some, all of them at -inf.
    float *po = nullptr;
    float2 *pml = nullptr;
    int pieces = 0;     // that paged_join_rows() adds
    int piece_out = -1; // >= 0: results go there as a piece instead of to `out`
    // Split ranges of paged_rows.cu: two pieces and one descriptor per CTA.
    float *ro = nullptr;
    float2 *rml = nullptr;
    int4 *meta = nullptr;
};

// fp32 values to the cache's type, rounded to nearest.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// 16 bytes to shared memory; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 2^x by the hardware's approximation (2 ulp; -inf gives 0).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a row's powers of two are taken against: its maximum `top` (in powers), less `by` in fp16, whose range of 2^15 above 1 would go unused
// otherwise.  Probabilities have all their digits down to 2^-14 then and a trace down to 2^-25, of what is 2^by now: with the maximum at
// 1, keys 17 nats below it would be lost from the sum of v while the sum of the powers has them, and 130 000 such keys are a part
// of the result that shows.  The sums with v and of the powers are scaled alike, in pieces too, since their m is this one.  (A large maximum
// is left as it is: the difference would be rounded.)
constexpr float kLargePower = 1048576.f;
template <typename T> __device__ __forceinline__ float lifted(float top, float by) {
    return std::is_same<T, __half>::value && fabsf(top) < kLargePower ? top - by : top;
}

// Attention of a's tokens over their keys (and the shared ones before them); *need: the workspace that it takes, all that is done where
// a.q is NULL.  Where n_prefix > 0, the same launch also forms `n_prefix` pieces of all tokens against a.s.n0 shared keys alone (one
// sequence of all tokens), and the sequences' own keys go without them.
int paged_rows_run(petb200_ctx *ctx, int dtype, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int n_prefix, cudaStream_t s);
// The same in 128-row tiles, 16-bit types.  pieces_out > 0: into so many pieces of the keys.
int paged_tiles_run(petb200_ctx *ctx, int dtype, PagedArgs a, char *ws, size_t ws_bytes, size_t *need, int pieces_out, cudaStream_t s);
// Pieces of the keys that paged_tiles_run() makes of a call by itself.
int paged_tiles_pieces(petb200_ctx *ctx, const PagedArgs &a);
// Adds each row's a.pieces pieces.
int paged_join_rows(petb200_ctx *ctx, int dtype, const PagedArgs &a, cudaStream_t s);

} // namespace petb200
