"""GPU: attention over a paged cache where numbers leave the ordinary range: infinities in keys and
values that every row sees, very large scores, and
probabilities that 16-bit types hold badly."""
import math

import pytest
import torch

from paged_oracle import HALF_STEP, Case

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ALL = [F32, F16, BF16]

# (new tokens of each sequence, query heads of a key head): one row, a few, most of a 16-row tile, several tiles of 16 and of 128
ROWS = [([1, 1], 1), ([4, 1], 1), ([1, 1], 5), ([1, 1], 16), ([3, 2], 2), ([40, 7], 5), ([150], 2)]


def place(c, b, key):
    return c.table[b, key // c.page].long(), key % c.page


def infinite_case(dtype, new, group, dim, planted, lens=(211, 333)):
    """A case with queries that 11 bits hold (as after a cast from bf16), and where key `planted` of each sequence lies."""
    c = Case(dtype, new, list(lens[:len(new)]), 2, group, dim, 1, device="cuda")
    c.q = c.q.to(BF16).to(dtype)
    return c, [place(c, b, planted) for b in range(len(new))]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("new,group", ROWS)
@pytest.mark.parametrize("dim", [40, 128])
@pytest.mark.parametrize("planted", [0, 3, 37])
def test_a_key_that_scores_minus_infinity_weighs_nothing(ctx, dtype, new, group, dim, planted):
    """-inf in a key, a positive query value against it: the result is that of the sequence without the key."""
    c, places = infinite_case(dtype, new, group, dim, planted)
    c.q[:, :, 5] = c.q[:, :, 5].abs() + 0.5
    for p in places:
        c.k[p][0, 5] = -math.inf  # the first key head's; the second one's stays a number
    got = c.attend(ctx).double().cpu()
    ctx.sync_check()
    assert torch.isfinite(got).all()
    for p in places:  # (any number will do for the second head's rows)
        c.k[p][0, 5] = 0
    want, tol = c.want()
    assert ((got[:, group:] - want[:, group:]).abs() <= tol[:, group:]).all()
    table = c.table
    c.table = torch.cat((table[:, :planted], table[:, planted + 1:]), 1)  # pages of one key: the key leaves with its page
    c.lens = [n - 1 for n in c.lens]
    want, tol = c.want()
    assert ((got[:, :group] - want[:, :group]).abs() <= tol[:, :group]).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("new,group", ROWS)
@pytest.mark.parametrize("dim", [40, 128])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_infinite_values_that_are_seen_are_the_result(ctx, dtype, new, group, dim, bad):
    """An infinity in v at two keys, one of them the key with the largest score: that column is infinite, all others as without it."""
    c, places = infinite_case(dtype, new, group, dim, 3)
    for b, p in enumerate(places):
        c.k[p][0] = c.q[c.starts[b], 0] / 4  # (along the first row's query: a probability near 1 there)
    want, tol = c.want()
    for b, p in enumerate(places):
        c.v[p][0, 7] = bad
        c.v[place(c, b, 100)][0, 7] = bad
        c.v[place(c, b, 50)][1, dim - 1] = -bad
    got = c.attend(ctx).double().cpu()
    ctx.sync_check()
    assert (got[:, :group, 7] == bad).all() and (got[:, group:, dim - 1] == -bad).all()
    plain = torch.ones_like(want, dtype=torch.bool)
    plain[:, :group, 7] = plain[:, group:, dim - 1] = False
    assert ((got - want).abs() <= tol)[plain].all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("new,group", ROWS)
def test_scores_and_values_without_an_answer_are_nan(ctx, dtype, new, group):
    """A score of +inf (inf - inf in the softmax), infinities of both signs in a column, a NaN in a key: NaN there and nowhere else."""
    c, places = infinite_case(dtype, new, group, 64, 3)
    want, tol = c.want()
    for b, p in enumerate(places):
        c.v[p][1, 7], c.v[place(c, b, 50)][1, 7] = math.inf, -math.inf
    got = c.attend(ctx).double().cpu()
    assert torch.isnan(got[:, group:, 7]).all()
    plain = torch.ones_like(want, dtype=torch.bool)
    plain[:, group:, 7] = False
    assert ((got - want).abs() <= tol)[plain].all()
    for number in (math.inf, math.nan):
        c.q[:, :, 9] = c.q[:, :, 9].abs() + 0.5
        for p in places:
            c.k[p][0, 9] = number
        got = c.attend(ctx)
        assert torch.isnan(got[:, :group]).all() and torch.isfinite(got[:, group:, :7]).all()
    ctx.sync_check()


@pytest.mark.parametrize("dtype,scale", [(F32, 1.0), (F32, 2.0 ** 12), (F16, 0.3), (F16, 11.0), (F16, 2.0 ** 12), (BF16, 0.3), (BF16, 11.0), (BF16, 2.0 ** 12)])
@pytest.mark.parametrize("new,lens,prefix", [([1], [400], 0), ([40, 150], [300, 2600], 0), ([3, 1], [90, 5], 700), ([60, 70], [60, 300], 700)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_many_millions_choose_a_key(ctx, dtype, scale, new, lens, prefix, sign):
    """Scores 2^20 * scale and more apart, far more than what 32 bits round at their size: each row is the value of the key that it scores highest."""
    c = Case(dtype, new, lens, 1, 2, 64, 16, prefix=prefix, device="cuda", garbage=False)
    c.q[:], c.k[:] = 0, 0
    c.q[:, 0, 0], c.q[:, 1, 0] = 2.0 ** 15, 2.0 ** 15 * 1.25
    places = [(c.prefix_table[j // 16].long(), j % 16) for j in range(prefix)]
    order = torch.randperm(prefix + max(lens), generator=torch.Generator().manual_seed(2)) % 128  # (several keys have the largest score)
    for j, (page, slot) in enumerate(places):
        c.k[page, slot, 0, 0] = sign * 32.0 * (1 + order[j])
    for b in range(len(lens)):
        for j in range(lens[b]):
            page, slot = place(c, b, j)
            c.k[page, slot, 0, 0] = sign * 32.0 * (1 + order[prefix + j])
    got = c.attend(ctx, scale=scale).double().cpu()
    ctx.sync_check()
    for b in range(len(lens)):
        k, v = c.keys(b, c.k)[:, 0, 0], c.keys(b, c.v)[:, 0]
        for i in range(new[b]):
            n = prefix + lens[b] - new[b] + i + 1
            top = k[:n] == k[:n].max()
            # probabilities are equal and exact but for a rounding to the type, which the sum does not have; the sum and mean of few keys
            want, tol = v[:n][top].mean(0), v[:n][top].abs().mean(0) * (2 * HALF_STEP[dtype] + 2.0 ** -17)
            assert ((got[c.starts[b] + i] - want).abs() <= tol).all(), (b, i)


# ---- probabilities far below the largest one -------------------------------------------------------------------------------------
def level_case(dtype, new, lens, top, gap, heads=1, group=1, page=64, prefix=0, **more):
    """All keys score 0 but key top(b) of each sequence (of the prefix where there is one), which scores `gap` and has v = 0; v = 1 elsewhere."""
    c = Case(dtype, new, lens, heads, group, 8, page, prefix=prefix, device="cuda", **more)
    c.q[:], c.k[:], c.v[:] = 0, 0, 1
    c.q[:, :, 0] = 1
    for b in range(len(lens)):
        if prefix:
            j = top(prefix)
            p = c.prefix_table[j // page].long(), j % page
        else:
            j = top(lens[b])
            p = place(c, b, j)
        c.k[p][:, 0], c.v[p] = gap, 0
    return c


def check_level(c, got, gap):
    """n keys of probability e^-gap beside one of 1.  A probability has a half step of the type relative to itself, or, in fp16, 2^-32 of the
    row's largest one where that is more (subnormal steps are 2^-24 of values scaled to 2^7 at least); the sum has n / 4 + 64 additions
    of 32 bits; the power's argument is rounded at gap * log2(e) and the product before it; the result to its type."""
    u, e = HALF_STEP[c.dtype], math.exp(-gap)
    for b, n in enumerate(c.lens):
        n += c.prefix - 1
        want = n * e / (1 + n * e)
        tol = want * (u + u + (n / 4 + 64) * 2.0 ** -24 + 4 * gap * 2.0 ** -23 + 2.0 ** -20) + n * 2.0 ** -32 + 2.0 ** -25
        off = (got[c.starts[b]:c.starts[b + 1]].double().cpu() - want).abs().max()
        assert off <= tol, f"{float(off):.3g} off {want:.3g}, {tol:.3g} allowed"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [9.0, 12.0, 15.0, 16.5, 17.5])
@pytest.mark.parametrize("top", [lambda n: 0, lambda n: n - 1, lambda n: n // 2], ids=["first", "last", "middle"])
# clusters, whole units, ranges, draft tokens on very many keys; tiles, tiles split over the keys
@pytest.mark.parametrize("new,lens,group", [([1], [3000], 1), ([1] * 3000, [250] * 3000, 1), ([1], [130000], 4), ([4, 4], [60000, 130000], 2),
                                            ([200], [9000], 1), ([30], [130000], 1)])
def test_keys_far_below_the_largest_keep_their_weight(ctx, dtype, gap, top, new, lens, group):
    c = level_case(dtype, new, lens, top, gap, group=group, starts=False, garbage=False)
    got = c.attend(ctx, causal=False, scale=1.0)
    ctx.sync_check()
    check_level(c, got, gap)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [12.0, 16.5, 17.5])
# a few rows (prefix and own keys in one launch), rows enough for tiles of the prefix, sequences that read it alone
@pytest.mark.parametrize("seqs,new,own,group", [(3, 1, 500, 1), (40, 1, 300, 4), (4, 60, 2000, 4)])
def test_keys_far_below_the_largest_behind_a_prefix(ctx, dtype, gap, seqs, new, own, group):
    c = level_case(dtype, [new] * seqs, [own] * seqs, lambda n: n // 3, gap, group=group, prefix=9000, starts=False, garbage=False)
    got = c.attend(ctx, causal=False, scale=1.0)
    ctx.sync_check()
    check_level(c, got, gap)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new", [1, 130])
@pytest.mark.parametrize("grows", [5.5, 5.625, 30.0])  # 2^8 is e^5.545: just within what the tiles let a maximum grow, just beyond, far beyond
def test_a_maximum_that_grows_stays_within_the_type(ctx, dtype, new, grows):
    """Half of the keys score `grows` above the other half, which come first: probabilities of the type's range until the maximum moves."""
    c = Case(dtype, [new], [2000], 1, 1, 8, 16, device="cuda", garbage=False)
    c.q[:], c.k[:], c.v[:] = 0, 0, 1
    c.q[:, :, 0] = 1
    for j in range(1000, 2000):
        p = place(c, 0, j)
        c.k[p][:, 0], c.v[p] = grows, 2
    c.check(c.attend(ctx, causal=False, scale=1.0), causal=False, scale=1.0)
    ctx.sync_check()
