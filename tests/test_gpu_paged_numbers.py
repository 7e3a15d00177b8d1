"""GPU: attention over a paged cache where numbers leave the ordinary range: infinities in keys and
values that every row sees, and very large scores."""
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
