"""GPU: the paged cache and the attentions that read it, against plain forms in 64 bits with tolerances derived from the arithmetic."""
import math

import pytest
import torch

from paged_oracle import HALF_STEP, Case, rotated
from pet_b200.lib import ERR_DEVICE, ERR_INVALID, ERR_UNSUPPORTED, PetError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ALL = [F32, F16, BF16]


# ---- appending ---------------------------------------------------------------------------------------------------------------
def append_case(ctx, dtype, source, new, lens, heads, q_heads, dim, page, pairs, interleaved, pos0=0, merged=True, layout="slots", behind=2, shift=0):
    c = Case(dtype, new, lens, heads, 1, dim, page, layout=layout, device="cuda", behind=behind, garbage=False)
    g = torch.Generator().manual_seed(5)
    total = q_heads + 2 * heads
    x = torch.randn(c.tokens, total, dim + shift, generator=g).to(source).cuda()[:, :, shift:]  # shift: rows off the 16-byte grid
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    if not merged:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float()
    kc, vc = c.pool(c.k), c.pool(c.v)
    q_out = torch.full((c.tokens, q_heads, dim), 7.0, dtype=dtype, device="cuda") if q_heads else None
    got = ctx.kv_append(k, v, kc, vc, c.on(c.table), c.on(torch.tensor(lens, dtype=torch.int32)), q_starts=c.on(c.q_starts), q=q if q_heads else None,
                        q_out=q_out, inv_freq=freq.cuda() if pairs else None, interleaved=interleaved, pos0=pos0)
    ctx.sync_check()
    assert got is q_out
    want_k, want_v, u = c.k.double(), c.v.clone(), HALF_STEP[dtype]
    tol_k = torch.zeros_like(want_k)
    q, k, v = (t.cpu() for t in (q, k, v))
    for b in range(len(lens)):
        for i in range(new[b]):
            p, row = lens[b] - new[b] + i, c.starts[b] + i
            angle = [(pos0 + p) * float(f) for f in freq]
            if q_heads:
                want, size = rotated(q[row], angle, interleaved)
                # fp32 products, sums and turns: cos and sin within 2^-22 of the angle's 2 pi * 2^-25 and their own rounding
                assert ((got[row].double().cpu() - want).abs() <= size * 2.0 ** -21 + want.abs() * u * 1.001 + 2.0 ** -25 * (dtype is F16)).all()
            if p < 0:
                continue
            page, slot = c.table[b, p // c.page].long(), p % c.page
            want, size = rotated(k[row], angle, interleaved)
            want_k[page, slot] = want
            tol_k[page, slot] = size * 2.0 ** -21 + want.abs() * u * 1.001 + 2.0 ** -25 * (dtype is F16)
            want_v[page, slot] = v[row].to(dtype)
    assert ((kc.double().cpu() - want_k).abs() <= tol_k).all()  # (rows that nobody appends to: unchanged to the bit)
    assert torch.equal(vc.cpu(), want_v)
    if q_heads:
        assert (got[c.starts[-1]:] == 7).all(), "rows behind the last sequence were written"


@pytest.mark.parametrize("dtype,source", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("dim,pairs,interleaved", [(128, 64, False), (128, 32, True), (64, 0, False), (80, 40, False), (40, 10, False), (8, 1, True), (8, 3, False)])
def test_append_turns_and_stores(ctx, dtype, source, dim, pairs, interleaved):
    append_case(ctx, dtype, source, [1, 3, 0, 5], [1, 40, 9, 17], 2, 4, dim, 16, pairs, interleaved)


@pytest.mark.parametrize("page", [1, 7, 64])
@pytest.mark.parametrize("layout", ["slots", "heads", "gaps"])
def test_append_to_any_page_and_layout(ctx, page, layout):
    append_case(ctx, BF16, BF16, [9, 2], [9, 130], 3, 3, 64, page, 32, False, layout=layout, merged=False)


def test_append_of_more_than_a_block_takes_and_without_queries(ctx):
    append_case(ctx, F16, F16, [700, 900, 1], [700, 901, 1], 2, 0, 64, 16, 32, False)
    append_case(ctx, BF16, F32, [1200], [1200], 1, 40, 64, 32, 32, True)


def test_many_sequences_of_uneven_prompts(ctx):
    """More sequences than are looked at together: rows find theirs, with empty ones among them."""
    new = [(3, 0, 1, 2)[b % 4] for b in range(2600)]
    append_case(ctx, BF16, BF16, new, [n + b % 3 for b, n in enumerate(new)], 1, 1, 8, 4, 4, False)
    new = [(17, 33, 0, 20)[b % 4] for b in range(150)]
    c = Case(BF16, new, [n + b % 50 for b, n in enumerate(new)], 1, 4, 64, 16, device="cuda")
    c.check(c.attend(ctx))
    c = Case(F16, [20] * 70, [20 + b for b in range(70)], 2, 4, 64, 16, device="cuda", starts=False)
    c.check(c.attend(ctx))
    ctx.sync_check()


def test_append_at_far_positions(ctx):
    """Angles of positions past 2^24: an fp32 product of position and frequency would be off by whole radians."""
    append_case(ctx, F32, F32, [3, 1], [5, 1], 1, 2, 64, 16, 32, False, pos0=2 ** 31 - 100)


@pytest.mark.parametrize("shift", [1, 2])
def test_append_from_rows_off_the_grid(ctx, shift):
    append_case(ctx, F16, F16, [2, 4], [2, 20], 2, 2, 64, 16, 32, False, shift=shift)
    append_case(ctx, BF16, F32, [2, 4], [2, 20], 2, 2, 64, 16, 32, True, shift=shift)


def test_append_with_more_tokens_than_keys_stores_the_last(ctx):
    append_case(ctx, F32, F32, [5, 4], [2, 0], 1, 1, 64, 16, 32, False)


# ---- attention over pages ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (3, 5), (1, 17)])
def test_single_tokens(ctx, dtype, dim, heads, group):
    c = Case(dtype, [1] * 6, [1, 2, 15, 64, 65, 333], heads, group, dim, device="cuda", starts=False)
    c.check(c.attend(ctx))
    ctx.sync_check()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("page,layout", [(1, "slots"), (7, "heads"), (16, "gaps"), (128, "slots")])
def test_pages_of_any_size_and_layout(ctx, dtype, page, layout):
    c = Case(dtype, [1, 2, 3], [130, 257, 3], 2, 2, 64, page, layout=layout, device="cuda", behind=3)
    out = torch.full_like(c.q, 5.0).cuda()
    c.check(c.attend(ctx, out=out))
    assert (out[c.starts[-1]:] == 5).all(), "rows behind the last sequence were written"
    ctx.sync_check()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens", [([33], [33]), ([5, 0, 70, 1], [5, 7, 200, 1]), ([130, 3], [131, 300]), ([257], [600])])
def test_prompts(ctx, dtype, causal, new, lens):
    for dim, heads, group in ((64, 1, 3), (128, 2, 1)):
        c = Case(dtype, new, lens, heads, group, dim, device="cuda")
        c.check(c.attend(ctx, causal=causal), causal=causal)
    ctx.sync_check()


@pytest.mark.parametrize("dtype", ALL)
def test_rows_that_see_nothing_give_zeros(ctx, dtype):
    c = Case(dtype, [1, 4, 1, 200], [0, 2, 5, 90], 2, 2, 64, device="cuda")
    got = c.attend(ctx)
    c.check(got)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[6:6 + 110] == 0).all()
    ctx.sync_check()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("new", [4, 300])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_keys_never_contribute(ctx, dtype, new, bad):
    """The newest key holds no number: rows before it are as if it were not there, its own row has the formula's NaN or infinity."""
    c = Case(dtype, [new], [new + 30], 1, 2, 64, device="cuda")
    at = new + 29
    page, slot = c.table[0, at // c.page].long(), at % c.page
    want, tol = c.want()
    c.v[page, slot, 0, 5] = bad
    got = c.attend(ctx).double().cpu()
    assert ((got[:-1] - want[:-1]).abs() <= tol[:-1]).all()
    assert (torch.isnan(got[-1, :, 5]) if math.isnan(bad) else got[-1, :, 5] == bad).all()
    keep = [d for d in range(64) if d != 5]
    assert ((got[-1][:, keep] - want[-1][:, keep]).abs() <= tol[-1][:, keep]).all()
    c.k[page, slot, 0, 3] = math.nan
    got = c.attend(ctx).double().cpu()
    assert ((got[:-1] - want[:-1]).abs() <= tol[:-1]).all() and torch.isnan(got[-1]).all()


@pytest.mark.parametrize("new,group", [(1, 1), (4, 1), (2, 2), (1, 3)])
@pytest.mark.parametrize("dim", [8, 64, 104, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_few_rows_in_full_precision(ctx, new, group, dim, bad):
    """Up to four rows of fp32: lengths around a warp's and a block's step, and newest keys that hold no numbers."""
    c = Case(F32, [new] * 9, [max(n, new) for n in (1, 7, 8, 9, 31, 33, 130, 700, 2050)], 2, group, dim, 16, device="cuda", starts=False)
    c.check(c.attend(ctx))
    if new > 1:
        want, tol = c.want()
        for b in range(9):
            at = c.lens[b] - 1
            c.v[c.table[b, at // c.page].long(), at % c.page, 1, 3] = bad
            c.k[c.table[b, at // c.page].long(), at % c.page, 0, 2] = bad
        got = c.attend(ctx).double().cpu()
        for b in range(9):
            rows, last = slice(c.starts[b], c.starts[b + 1] - 1), c.starts[b + 1] - 1
            assert ((got[rows] - want[rows]).abs() <= tol[rows]).all()
            assert not torch.isfinite(got[last, group:, 3]).any() and (torch.isnan(got[last, :group]).all() or bad == math.inf)
    ctx.sync_check()


@pytest.mark.parametrize("dtype", ALL)
def test_long_sequences_among_short_ones(ctx, dtype):
    """Ranges of work that cut a sequence many times, and take many sequences whole."""
    c = Case(dtype, [1] * 40, [9000] + [3] * 38 + [2500], 2, 4, 64, 16, device="cuda", starts=False)
    c.check(c.attend(ctx))
    c = Case(dtype, [4], [20001], 1, 4, 128, 64, device="cuda")
    c.check(c.attend(ctx))


# Few sequences on a cluster of eight blocks each, more on four, more on ranges: keys that leave some blocks of a cluster without any, none at all
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("seqs", [1, 20, 40, 80])
@pytest.mark.parametrize("dim", [64, 104])
def test_sequences_that_share_the_gpu(ctx, dtype, seqs, dim):
    lens = [(0, 1, 63, 64, 65, 300, 511, 900)[b % 8] for b in range(seqs)]
    if seqs == 1:
        lens = [700]
    c = Case(dtype, [1 + b % 2 for b in range(seqs)], [max(n, 0) for n in lens], 2, 5, dim, 16, device="cuda", behind=2, seed=seqs)
    out = torch.full_like(c.q, 5.0).cuda()
    c.check(c.attend(ctx, out=out))
    assert (out[c.starts[-1]:] == 5).all()
    ctx.sync_check()


def test_many_short_sequences(ctx):
    c = Case(BF16, [1] * 700, [1 + b % 37 for b in range(700)], 4, 2, 64, 16, device="cuda", starts=False)
    c.check(c.attend(ctx))


@pytest.mark.parametrize("dtype", ALL)
def test_large_scores_and_a_scale(ctx, dtype):
    """Scores in the hundreds: one key takes all; the maximum arrives late and early."""
    c = Case(dtype, [1, 70], [150, 170], 2, 2, 64, device="cuda")
    c.q *= 8
    c.check(c.attend(ctx, scale=0.5), scale=0.5)


# Rows around a tile of 128 and a pair of tiles, keys around a tile of 128, heads narrower than the tile's 64 or 128 columns
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("rows,keys", [(64, 64), (127, 127), (128, 128), (129, 129), (255, 400), (256, 256), (257, 513)])
def test_tiles_of_rows_and_keys(ctx, dtype, dim, rows, keys):
    c = Case(dtype, [rows], [keys], 1, 1, dim, 16, device="cuda")
    c.check(c.attend(ctx))
    ctx.sync_check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,lens,heads,group", [([100], [6100], 1, 1), ([40, 30], [3000, 31], 2, 5), ([64, 1, 200], [2000, 2500, 200], 1, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows_on_many_keys_are_split(ctx, dtype, new, lens, heads, group, causal):
    for layout, page in (("heads", 64), ("gaps", 9)):
        c = Case(dtype, new, lens, heads, group, 64, page, layout=layout, device="cuda", behind=4)
        out = torch.full_like(c.q, 5.0).cuda()
        c.check(c.attend(ctx, causal=causal, out=out), causal=causal)
        assert (out[c.starts[-1]:] == 5).all()


# Pages that are boxes of a tile, hold several tiles, or fit neither; shared keys that end inside a tile and inside a page
@pytest.mark.parametrize("page", [1, 8, 24, 32, 128, 256, 200])
@pytest.mark.parametrize("layout", ["slots", "heads", "gaps"])
@pytest.mark.parametrize("prefix", [0, 75, 700])
def test_tiles_over_pages_of_any_size(ctx, page, layout, prefix):
    c = Case(BF16, [70, 0, 140], [70, 9, 560], 2, 2, 128 if page == 32 else 72, page, prefix=prefix, layout=layout, device="cuda")
    c.check(c.attend(ctx))
    ctx.sync_check()


def test_pools_of_one_page_and_of_one_head_for_all(ctx):
    """Strides of extents of one are never used; an expanded pool (stride 0) is read as it is."""
    c = Case(F16, [70], [100], 1, 2, 64, 128, device="cuda")
    k, v = c.pool(c.k), c.pool(c.v)
    odd = [t.as_strided(t.shape, (t.stride(0), t.stride(1), 3, 1)) for t in (k, v)]
    t, n = c.on(c.table), torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    c.check(ctx.attention_paged(c.on(c.q), *odd, t, n, q_starts=c.on(c.q_starts)))
    for new in (70, 1):
        c = Case(F16, [new], [100], 1, 2, 64, 128, device="cuda")
        c.check(ctx.attention_paged(c.on(c.q), *(c.pool(x).expand(-1, -1, 2, -1) for x in (c.k, c.v)), c.on(c.table), n, q_starts=c.on(c.q_starts)))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_maximum_that_grows_late(ctx, dtype):
    """Scores that rise along the keys by far more than the sums' range allows without scaling, and rows that stay at one level."""
    c = Case(dtype, [130], [900], 1, 1, 64, device="cuda")
    for j in range(900):
        page, slot = c.table[0, j // c.page].long(), j % c.page
        c.k[page, slot] = (torch.randn(1, 64) * 0.1 + j / 100).to(dtype)
    c.q[:60] = c.q[:60].abs()
    c.q[60:90] = 0
    c.check(c.attend(ctx))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_values_in_split_tiles(ctx, bad):
    """Non-finite values of v among the newest keys, where the keys are split over blocks: only the rows that see them have them."""
    c = Case(BF16, [100], [3000], 1, 1, 64, device="cuda")
    want, tol = c.want()
    for at, d in ((2950, 5), (2999, 9), (2925, 63)):
        c.v[c.table[0, at // c.page].long(), at % c.page, 0, d] = bad
    got = c.attend(ctx).double().cpu()
    seen = {5: 50, 9: 99, 63: 25}
    for d in range(64):
        clean = seen.get(d, 100)
        assert ((got[:clean, 0, d] - want[:clean, 0, d]).abs() <= tol[:clean, 0, d]).all()
        assert not torch.isfinite(got[clean:, 0, d]).any()


def test_strided_queries_and_output(ctx):
    c = Case(BF16, [3, 70], [90, 70], 2, 3, 64, device="cuda")
    wide = torch.randn(c.tokens, 10, 64, device="cuda").to(BF16)
    wide[:, 2:8] = c.q.cuda()
    out = torch.full((c.tokens, 9, 64), 3.0, device="cuda", dtype=BF16)
    c.attend(ctx, q=wide[:, 2:8], out=out[:, 1:7])
    c.check(out[:, 1:7])
    assert (out[:, 0] == 3).all() and (out[:, 7:] == 3).all()
    odd = torch.zeros(c.tokens, 6, 65, device="cuda", dtype=BF16)  # rows off the 16-byte grid
    odd[:, :, :64] = c.q.cuda()
    c.check(c.attend(ctx, q=odd[:, :, :64]))


# ---- a shared prefix ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("prefix", [1, 16, 333, 1500])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 40, 0]), ([2, 5, 1], [2, 70, 9]), ([80, 0, 33], [80, 3, 100]), ([1], [12])])
def test_prefix(ctx, dtype, prefix, new, lens):
    for dim, heads, group, page in ((64, 2, 3, 16), (128, 1, 8, 7)):
        c = Case(dtype, new, lens, heads, group, dim, page, prefix=prefix, device="cuda", behind=1)
        out = torch.full_like(c.q, 5.0).cuda()
        c.check(c.attend(ctx, out=out))
        assert (out[c.starts[-1]:] == 5).all()
    ctx.sync_check()


def test_prefix_of_many_sequences_and_of_no_keys(ctx):
    c = Case(BF16, [1] * 50, [1 + 3 * b for b in range(50)], 2, 4, 128, 16, prefix=2100, device="cuda", starts=False)
    c.check(c.attend(ctx))
    c = Case(F16, [1] * 5, [1 + 3 * b for b in range(5)], 2, 4, 64, 16, prefix=0, device="cuda", starts=False)
    got = ctx.attention_prefix(c.on(c.q), c.pool(c.k), c.pool(c.v), torch.empty(0, dtype=torch.int32, device="cuda"), 0, c.on(c.table),
                               torch.tensor(c.lens, dtype=torch.int32, device="cuda"))
    c.check(got)


# ---- together, captured, beside each other ----------------------------------------------------------------------------------------
def test_a_step_of_a_decoder_layer(ctx):
    """Projection -> append -> attention, token by token, against attention over the same keys kept densely."""
    g = torch.Generator().manual_seed(3)
    heads, group, dim, page, steps = 2, 2, 64, 16, 40
    width = (heads * group + 2 * heads) * dim
    w = (torch.randn(128, width, generator=g) / 128 ** 0.5).cuda()
    kc, vc = torch.zeros(16, page, heads, dim, device="cuda"), torch.zeros(16, page, heads, dim, device="cuda")
    table = torch.tensor([[3, 9, 1], [0, 14, 7]], dtype=torch.int32, device="cuda")
    freq = (10000.0 ** (-torch.arange(32) / 32)).cuda()
    dense_k, dense_v = [], []
    for t in range(steps):
        x = torch.randn(1, 2, 128, generator=g).cuda()
        lens = torch.tensor([t + 1, t + 1], dtype=torch.int32, device="cuda")
        qkv = ctx.matmul(x, w[None])[0].view(2, -1, dim)
        q = ctx.kv_append(qkv[:, 4:6], qkv[:, 6:], kc, vc, table, lens, q=qkv[:, :4], inv_freq=freq)
        y = ctx.attention_paged(q, kc, vc, table, lens)
        raw = qkv.cpu().double()
        ang = [t * float(f) for f in freq.cpu()]
        dense_k.append(torch.stack([rotated(raw[b, 4:6], ang, False)[0] for b in range(2)]))
        dense_v.append(raw[:, 6:])
        qq = torch.stack([rotated(raw[b, :4], ang, False)[0] for b in range(2)])
        kk, vv = torch.stack(dense_k, 1).repeat_interleave(2, 2), torch.stack(dense_v, 1).repeat_interleave(2, 2)
        p = torch.softmax(torch.einsum("bhd,bnhd->bhn", qq, kk) * dim ** -0.5, -1)
        want = torch.einsum("bhn,bnhd->bhd", p, vv)
        # turns of 2^-21 on q and k move a score of at most ~8 by 2^-17; the rest is smaller
        assert (y.cpu().double() - want).abs().max() <= 2.0 ** -16 * float(vv.abs().max())
    ctx.sync_check()


def test_captured_call_reads_new_lengths(ctx):
    c = Case(BF16, [1] * 4, [50, 1, 200, 90], 2, 4, 64, device="cuda", starts=False, width=20)
    q, k, v, t = c.on(c.q), c.pool(c.k), c.pool(c.v), c.on(c.table)
    lens = torch.tensor([10, 1, 3, 90], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    ctx.attention_paged(q, k, v, t, lens, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.attention_paged(q, k, v, t, lens, out=out)
    lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    c.check(out)


def test_captured_layer_with_a_prefix(ctx):
    """Append, attention behind a prefix and attention of prompts in one graph, replayed on other inputs and lengths."""
    heads, dim, page, prefix = 2, 64, 16, 100
    g = torch.Generator().manual_seed(9)
    kc, vc = (torch.randn(60, page, heads, dim, generator=g).to(BF16).cuda() for _ in "kv")
    table = torch.arange(60, dtype=torch.int32)[10:58].view(3, 16).contiguous().cuda()
    head = torch.arange(7, dtype=torch.int32).cuda()
    freq = (10000.0 ** (-torch.arange(32) / 32)).cuda()
    lens = torch.tensor([4, 9, 1], dtype=torch.int32, device="cuda")
    long, starts = torch.tensor([70, 90, 80], dtype=torch.int32, device="cuda"), torch.tensor([0, 70, 130, 200], dtype=torch.int32, device="cuda")
    x, p = torch.zeros(3, 8, dim, device="cuda", dtype=BF16), torch.zeros(200, 4, dim, device="cuda", dtype=BF16)

    def layer():
        q = ctx.kv_append(x[:, 4:6], x[:, 6:], kc, vc, table, lens, q=x[:, :4], inv_freq=freq, pos0=prefix)
        return q, ctx.attention_prefix(q, kc, vc, head, prefix, table, lens), ctx.attention_paged(p, kc, vc, table, long, q_starts=starts)
    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    x.copy_(torch.randn(3, 8, dim, generator=g).to(BF16))
    p.copy_(torch.randn(200, 4, dim, generator=g).to(BF16))
    lens.copy_(torch.tensor([40, 1, 200], dtype=torch.int32))
    long.copy_(torch.tensor([200, 60, 70], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    replayed = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(replayed, layer()))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(replayed, got))


def test_calls_on_two_streams(ctx):
    """Workspaces are a call's own: calls that overlap give what they give alone."""
    cases = [Case(F16, [1] * 8, [700 + 31 * b for b in range(8)], 2, 4, 128, device="cuda", starts=False, seed=s, prefix=p) for s, p in ((1, 0), (2, 300))]
    args = [(c.on(c.q), c.pool(c.k), c.pool(c.v), c.on(c.prefix_table), c.on(c.table), torch.tensor(c.lens, dtype=torch.int32, device="cuda")) for c in cases]
    def call(i):
        q, k, v, pt, t, n = args[i]
        return ctx.attention_prefix(q, k, v, pt, cases[i].prefix, t, n) if cases[i].prefix else ctx.attention_paged(q, k, v, t, n)
    alone = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, alone[i]) for x in got[i]), "results depend on what runs beside the call"


def test_offsets_past_32_bits(ctx):
    """A cache of more than 2^31 elements: its last pages are read and written."""
    page, heads, dim = 64, 8, 128
    pages = 2 ** 31 // (page * heads * dim) + 40
    kc = torch.zeros(pages, page, heads, dim, device="cuda", dtype=BF16)
    vc = torch.zeros(pages, page, heads, dim, device="cuda", dtype=BF16)
    table = torch.tensor([[pages - 1, pages - 7, 5]], dtype=torch.int32, device="cuda")
    x = torch.randn(130, 3 * heads, dim, device="cuda").to(BF16)
    lens = torch.tensor([130], dtype=torch.int32, device="cuda")
    ctx.kv_append(x[:, heads:2 * heads], x[:, 2 * heads:], kc, vc, table, lens)
    assert torch.equal(kc[pages - 1], x[:64, heads:2 * heads]) and torch.equal(vc[pages - 7], x[64:128, 2 * heads:]) and torch.equal(vc[5, :2], x[128:, 2 * heads:])
    got = ctx.attention_paged(x[:, :heads], kc, vc, table, lens)
    c = Case(BF16, [130], [130], heads, 1, dim, page, device="cuda", garbage=False)
    rows = torch.stack([c.table[0, j // page].long() * page + j % page for j in range(130)])
    c.k.view(-1, heads, dim)[rows], c.v.view(-1, heads, dim)[rows], c.q = x[:, heads:2 * heads].cpu(), x[:, 2 * heads:].cpu(), x[:, :heads].cpu()
    c.check(got)


# ---- what the device finds wrong ----------------------------------------------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported(ctx):
    for new in (1, 40):
        c = Case(BF16, [new, new], [60, 80], 2, 2, 64, device="cuda", garbage=False)
        c.table[1, 2] = -5
        c.attend(ctx)
        with pytest.raises(PetError, match="page") as e:
            ctx.sync_check()
        assert e.value.status == ERR_DEVICE
        ctx.sync_check()  # told once
        c = Case(BF16, [new, new], [60, 80], 2, 2, 64, device="cuda", garbage=False)
        x = torch.ones(2 * new, 2, 64, device="cuda", dtype=BF16)
        lens = torch.tensor([60, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        ctx.attention_paged(c.on(c.q), c.pool(c.k), c.pool(c.v), c.on(c.table[:, :5]), lens, q_starts=c.on(c.q_starts))
        with pytest.raises(PetError, match="more keys"):
            ctx.sync_check()
        kc, vc = c.pool(c.k), c.pool(c.v)
        ctx.kv_append(x, x, kc, vc, c.on(c.table), lens, q_starts=c.on(c.q_starts))
        with pytest.raises(PetError, match="page"):
            ctx.sync_check()


def test_starts_out_of_order_reach_no_other_memory(ctx):
    c = Case(BF16, [2, 2], [60, 80], 2, 2, 64, device="cuda")
    starts = torch.tensor([-7, 900, 3], dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 4, 64, device="cuda", dtype=BF16)
    ctx.attention_paged(c.on(c.q), c.pool(c.k), c.pool(c.v), c.on(c.table), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), q_starts=starts, out=out)
    ctx.sync_check()
    assert torch.isfinite(out).all()


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_refused_by_the_library(ctx):
    c = Case(BF16, [1, 1], [20, 30], 2, 2, 64, device="cuda", starts=False)
    q, t, n = c.on(c.q), c.on(c.table), torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    k, v = c.pool(c.k), c.pool(c.v)

    def refused(status, call):
        with pytest.raises(PetError) as e:
            call()
        assert e.value.status == status
    for scale in (0.0, -1.0, math.inf, math.nan):
        refused(ERR_INVALID, lambda: ctx.attention_paged(q, k, v, t, n, scale=scale))
    refused(ERR_INVALID, lambda: ctx.attention_paged(q[:, :3], k, v, t, n))  # 3 query heads on 2
    refused(ERR_INVALID, lambda: ctx.attention_paged(q.repeat(2, 1, 1)[:3], k, v, t, n))  # 3 tokens of 2 sequences
    refused(ERR_UNSUPPORTED, lambda: ctx.attention_paged(q.repeat(1, 1, 4)[:, :, :136], *(torch.zeros(4, 16, 2, 136, device="cuda", dtype=BF16) for _ in "kv"), t, n))
    refused(ERR_UNSUPPORTED, lambda: ctx.attention_paged(q[:, :, :60].contiguous(), *(torch.zeros(4, 16, 2, 60, device="cuda", dtype=BF16) for _ in "kv"), t, n))
    odd = torch.zeros(4 * 16 * 2 * 64 + 8, device="cuda", dtype=BF16)[1:-7].view(4, 16, 2, 64)
    refused(ERR_UNSUPPORTED, lambda: ctx.attention_paged(q, odd, odd, t, n))
    refused(ERR_UNSUPPORTED, lambda: ctx.attention_paged(q, k, v, t, n, out=torch.zeros(2, 4, 65, device="cuda", dtype=BF16)[:, :, :64]))
    refused(ERR_UNSUPPORTED, lambda: ctx.kv_append(q[:, :2], q[:, 2:], odd, odd, t, n))
    refused(ERR_INVALID, lambda: ctx.kv_append(q[:, :2], q[:, 2:], k, v, t, n, inv_freq=torch.ones(33, device="cuda")))
    refused(ERR_INVALID, lambda: ctx.kv_append(q[:, :2], q[:, 2:], k, v, t, n, q=q, q_out=q))
    refused(ERR_INVALID, lambda: ctx.attention_paged(q, k[:0], v[:0], t, n))
    ctx.sync_check()
    for empty in (q[:0],):
        assert ctx.attention_paged(empty, k, v, t[:0], n[:0]).shape == (0, 4, 64)
        assert ctx.kv_append(empty[:, :2], empty[:, 2:], k, v, t[:0], n[:0]) is None
