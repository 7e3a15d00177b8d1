"""GPU: calls of the paged cache as the documentation allows them, at its edges: outputs beside and over inputs, empty calls."""
import pytest
import torch

from paged_oracle import Case
from pet_b200.lib import ERR_DEVICE, ERR_INVALID, PetError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def arguments(c):
    return c.pool(c.k), c.pool(c.v), c.on(c.table), torch.tensor(c.lens, dtype=torch.int32, device="cuda")


def test_empty_calls_with_outputs(ctx):
    c = Case(BF16, [1, 1], [20, 30], 2, 2, 64, device="cuda", starts=False)
    k, v, t, n = arguments(c)
    q, buf = c.on(c.q), torch.full((4, 4, 64), 3.0, device="cuda", dtype=BF16)
    none, before = q[:0], (k.clone(), v.clone())
    assert ctx.kv_append(none[:, :2], none[:, 2:], k, v, t[:0], n[:0], q=none, q_out=buf[:0]).shape == (0, 4, 64)
    assert ctx.attention_paged(none, k, v, t[:0], n[:0], out=buf[:0]).shape == (0, 4, 64)
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")  # sequences without tokens
    assert ctx.kv_append(none[:, :2], none[:, 2:], k, v, t, n, q_starts=starts, q=none, q_out=buf[:0]).shape == (0, 4, 64)
    assert ctx.attention_paged(none, k, v, t, n, q_starts=starts, out=buf[:0]).shape == (0, 4, 64)
    ctx.sync_check()
    assert (buf == 3).all() and all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip((k, v), before))


@pytest.mark.parametrize("new", [1, 40])
def test_outputs_beside_and_over_inputs(ctx, new):
    c = Case(BF16, [new, new], [60, 80], 2, 2, 64, device="cuda", starts=False)
    k, v, t, n = arguments(c)

    def refused(call):
        with pytest.raises(PetError, match="overlap") as e:
            call()
        assert e.value.status == ERR_INVALID
    both = torch.zeros(c.tokens + 1, 12, 64, device="cuda", dtype=BF16)
    q = both[:-1, :4]
    q.copy_(c.on(c.q))
    for out in (both[:-1, :4], both[:-1, 3:7], both[1:, :4], both[1:, 1:5], both.view(-1, 4, 64)[:c.tokens]):
        refused(lambda: ctx.attention_paged(q, k, v, t, n, out=out))
    c.check(ctx.attention_paged(q, k, v, t, n, out=both[:-1, 4:8]))  # side by side in each token
    c.check(ctx.attention_paged(q, k, v, t, n, out=both[1:, 8:12]))
    ctx.sync_check()
    # appending: queries, keys and values of a merged projection, the turned queries beside them
    for out in (both[:-1, :4], both[:-1, 3:7], both[:-1, 6:10], both[1:, 5:9]):
        refused(lambda: ctx.kv_append(both[:-1, 4:6], both[:-1, 6:8], k, v, t, n, q=q, q_out=out))
    got = ctx.kv_append(both[:-1, 4:6], both[:-1, 6:8], k, v, t, n, q=q, q_out=both[:-1, 8:])
    ctx.sync_check()
    assert torch.equal(got, q) and got.data_ptr() == both[:, 8:].data_ptr()
    wide = torch.zeros(c.tokens, 8, 64, device="cuda")  # fp32 sources, the queries' halves inside their memory
    refused(lambda: ctx.kv_append(wide[:, 4:6], wide[:, 6:], k, v, t, n, q=wide[:, :4], q_out=wide.view(BF16).view(c.tokens, 16, 64)[:, 12:]))


def hooks():
    import ctypes as C
    from pet_b200 import lib as L
    lib = L.load()
    lib.petb200_debug_set_wait_limit.argtypes = [C.c_ulonglong]
    lib.petb200_debug_paged_starve.argtypes = [C.c_void_p, C.c_int]
    lib.petb200_debug_conv_starve.argtypes = [C.c_void_p, C.c_int]
    return lib


# Keys by TMA and by copies, tiles that split their keys, the shared prefix in tiles; fewer keys than the ring's stages hold, and many more
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("new,lens,prefix", [([150, 40], [150, 300], 0), ([100], [5000], 0), ([1] * 40, [90] * 40, 2000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_wait_that_runs_out_is_reported(ctx, page, new, lens, prefix, dim):
    """A ring whose stages expect an arrival that never comes, waits of 5 ms: the call returns, says so once, and the next one is right."""
    import time
    lib = hooks()
    c = Case(BF16, new, lens, 1, 4, dim, page, prefix=prefix, device="cuda")
    c.check(c.attend(ctx))
    ctx.sync_check()
    assert lib.petb200_debug_set_wait_limit(5_000_000) == 0
    try:
        assert lib.petb200_debug_paged_starve(ctx.h, 1) == 0
        began = time.monotonic()
        c.attend(ctx)
        with pytest.raises(PetError, match="wait") as e:
            ctx.sync_check()
        assert e.value.status == ERR_DEVICE and time.monotonic() - began < 1.5  # (the unshortened wait is 2 s)
    finally:
        lib.petb200_debug_paged_starve(ctx.h, 0)
        assert lib.petb200_debug_set_wait_limit(2_000_000_000) == 0
    c.check(c.attend(ctx))
    ctx.sync_check()


@pytest.mark.parametrize("last", ["attention", "convolution"])
def test_a_bad_page_and_a_wait_that_runs_out_are_both_reported(ctx, last):
    lib = hooks()
    c = Case(BF16, [1, 1], [60, 80], 2, 2, 64, device="cuda", garbage=False)
    c.table[1, 2] = -5
    tiles = Case(BF16, [150], [150], 1, 2, 64, device="cuda")
    x, w = torch.randn(1, 64, 28, 28, device="cuda"), torch.randn(64, 64, 3, 3, device="cuda")
    plan = ctx.conv2d_plan(x.shape, w.shape, 1, 1)
    ctx.conv2d_set_weights(plan, w)
    assert lib.petb200_debug_set_wait_limit(5_000_000) == 0
    try:
        c.attend(ctx)
        if last == "attention":
            assert lib.petb200_debug_paged_starve(ctx.h, 1) == 0
            tiles.attend(ctx)
        else:
            assert lib.petb200_debug_conv_starve(plan.h, 1) == 0
            ctx.conv2d_run(plan, x)
        with pytest.raises(PetError, match="wait.*page") as e:
            ctx.sync_check()
        assert e.value.status == ERR_DEVICE
    finally:
        lib.petb200_debug_paged_starve(ctx.h, 0)
        lib.petb200_debug_conv_starve(plan.h, 0)
        assert lib.petb200_debug_set_wait_limit(2_000_000_000) == 0
    ctx.sync_check()


def told(ctx):
    """What the device has to say of the calls so far."""
    try:
        ctx.sync_check()
    except PetError as e:
        assert e.status == ERR_DEVICE
        return str(e)
    return ""


LARGE, SMALL = 2 ** 31 - 1, -2 ** 31
BAD_STARTS = [[-7, 900, 3, 4], [5, 2, 4, 1], [LARGE, SMALL, 3, LARGE], [0, LARGE, 0, LARGE], [SMALL, SMALL, SMALL, SMALL], [3, 3, 3, 2], [1, 0, 9, 0]]


# rows on a cluster, in ranges, as whole units; tiles, split and not; a prefix read together and alone
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,keys,group,prefix", [(2, 60, 2, 0), (3, 9000, 2, 0), (2, 40, 40, 0), (60, 300, 3, 0), (40, 5000, 2, 0), (2, 60, 2, 700), (80, 90, 2, 700)])
def test_bad_starts_reach_no_other_memory(ctx, dtype, new, keys, group, prefix):
    """Starts that run backwards or past the tokens: whatever the result, nothing outside the call's rows and the sequences' pages is written."""
    c = Case(dtype, [new] * 3, [keys] * 3, 2, group, 64, 16, prefix=prefix, device="cuda", garbage=False)
    k, v, t, n = arguments(c)
    before, named = (k.clone(), v.clone()), torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
    named[t[:, :-(-keys // 16)].flatten().long()] = True
    heads, rows = 2 * group, slice(3, 3 + c.tokens)
    big = [torch.full((c.tokens + 6, heads, 64), 7.0, dtype=dtype, device="cuda") for _ in range(3)]
    q, out, q_out = (b[rows] for b in big)
    q.copy_(c.on(c.q))
    for starts in BAD_STARTS:
        s = torch.tensor(starts, dtype=torch.int32, device="cuda")
        if prefix:
            ctx.attention_prefix(q, k, v, c.on(c.prefix_table), prefix, t, n, q_starts=s, out=out)
        else:
            ctx.attention_paged(q, k, v, t, n, q_starts=s, out=out)
        assert "page" not in told(ctx)
        ctx.kv_append(q[:, :2], q[:, 2:4], k, v, t, n, q_starts=s, q=q, q_out=q_out, inv_freq=torch.ones(16, device="cuda"), pos0=prefix)
        assert told(ctx) == ""
        for b in big:
            assert (b[:3] == 7).all() and (b[-3:] == 7).all()
        assert torch.equal(k[~named], before[0][~named]) and torch.equal(v[~named], before[1][~named])
    s = c.on(c.q_starts)  # the same memory, in order
    k.copy_(before[0]), v.copy_(before[1])
    c.check(c.attend(ctx))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,keys,group", [(8, 60, 8), (8, 9000, 4), (16, 40, 40), (300, 300, 2), (100, 5000, 4)])
def test_starts_that_claim_more_rows_than_there_are(ctx, dtype, new, keys, group):
    """Sequences that have the tokens of others too, more together than the call: told once, and the next call is right."""
    c = Case(dtype, [new] * 8, [keys] * 8, 1, group, 64, 16, device="cuda", garbage=False, width=-(-keys // 16))
    k, v, t, n = arguments(c)
    q = c.on(c.q)
    s = torch.tensor([0, c.tokens] * 4 + [0], dtype=torch.int32, device="cuda")
    ctx.attention_paged(q, k, v, t, n, q_starts=s)
    assert "q_starts" in told(ctx)
    assert told(ctx) == ""
    c.check(c.attend(ctx))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_a_single_token_or_head_are_never_used(ctx, dtype):
    c = Case(dtype, [1], [50], 2, 2, 64, device="cuda", starts=False)
    k, v, t, n = arguments(c)
    q, out, q_out = (torch.zeros(256, device="cuda", dtype=dtype).as_strided((1, 4, 64), (257, 64, 1)) for _ in range(3))
    q.copy_(c.on(c.q))
    assert ctx.attention_paged(q, k, v, t, n, out=out).data_ptr() == out.data_ptr()
    c.check(out)
    ctx.kv_append(q[:, :2], q[:, 2:], k, v, t, n, q=q, q_out=q_out)
    ctx.sync_check()
    assert torch.equal(q_out, q) and torch.equal(k[c.table[0, 3].long(), 1], q[0, :2])
    c = Case(dtype, [3, 3], [50, 60], 1, 1, 64, device="cuda", starts=False)
    k, v, t, n = arguments(c)
    q, out = (torch.zeros(6, 64, device="cuda", dtype=dtype).as_strided((6, 1, 64), (64, 3, 1)) for _ in range(2))
    q.copy_(c.on(c.q))
    c.check(ctx.attention_paged(q, k, v, t, n, out=out))
    ctx.sync_check()


def test_scales_past_what_powers_of_two_hold_are_refused(ctx):
    """3e38 is finite, its product with log2(e) is not: every score of 0 would be 0 x infinity."""
    c = Case(F32, [1], [50], 2, 2, 64, device="cuda", starts=False)
    c.q *= 1e-38
    for scale in (3e38, 2.4e38):
        with pytest.raises(PetError) as e:
            c.attend(ctx, scale=scale)
        assert e.value.status == ERR_INVALID
    c.q[:], c.k[:] = 0, 0
    got = c.attend(ctx, scale=2.3e38).double().cpu()  # all scores are 0: the mean of v
    want = c.keys(0, c.v).mean(0).repeat_interleave(2, 0)
    assert ((got[0] - want).abs() <= c.keys(0, c.v).abs().mean(0).repeat_interleave(2, 0) * 2.0 ** -18).all()
    ctx.sync_check()


# ---- routes that a call takes by its sizes ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
# a token of one and of several sequences, a few rows, a prompt; tables of 512 to 131072 keys
@pytest.mark.parametrize("new,lens,group", [([1], [1500], 4), ([1] * 24, [1 + 60 * b for b in range(24)], 4), ([4, 1], [1500, 3], 2), ([200], [700], 2)])
@pytest.mark.parametrize("width", [128, 4096])
def test_tables_much_wider_than_their_sequences(ctx, dtype, new, lens, group, width):
    c = Case(dtype, new, lens, 2, group, 64, 16, width=width, device="cuda", behind=1)
    out = torch.full_like(c.q, 5.0).cuda()
    c.check(c.attend(ctx, out=out))
    assert (out[c.starts[-1]:] == 5).all()
    ctx.sync_check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
# the prompt's rows go to 16-row tiles with the tokens, the tokens to the prompt's tiles
@pytest.mark.parametrize("singles,prompt", [(63, 200), (7, 600)])
@pytest.mark.parametrize("prefix", [0, 500])
def test_single_tokens_beside_a_prompt(ctx, dtype, singles, prompt, prefix):
    new = [1] * (singles // 2) + [prompt] + [1] * (singles - singles // 2)
    c = Case(dtype, new, [n + 37 * b % 900 for b, n in enumerate(new)], 1, 4, 64, 16, prefix=prefix, device="cuda", behind=2)
    out = torch.full_like(c.q, 5.0).cuda()
    c.check(c.attend(ctx, out=out))
    assert (out[c.starts[-1]:] == 5).all()
    ctx.sync_check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("starts", [True, False])
# rows of a sequence that go together with the others' against the shared keys: up to 191, and the first that go alone
@pytest.mark.parametrize("new,group,prefix", [(1, 4, 3000), (10, 4, 3000), (31, 2, 3000), (31, 2, 2950), (95, 2, 9300), (96, 2, 9300)])
def test_a_prefix_in_tiles_for_all_sequences(ctx, dtype, dim, starts, new, group, prefix):
    """The shared keys by TMA (pages that are boxes of a tile), in tiles that hold several sequences' rows."""
    c = Case(dtype, [new] * 20 if new < 90 else [new] * 3, [new + 9 * b for b in range(20 if new < 90 else 3)], 1, group, dim, 32, prefix=prefix, device="cuda", starts=starts)
    c.check(c.attend(ctx))
    ctx.sync_check()


@pytest.mark.parametrize("new,group", [(1, 1), (4, 1), (2, 2), (1, 3), (1, 4)])
@pytest.mark.parametrize("dim", [8, 64, 104, 128])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_infinities_in_few_rows_of_full_precision(ctx, new, group, dim, bad):
    """Up to four rows of fp32, the newest key infinite: the row that sees it has what the 64-bit form has, the rows before it are as without it."""
    c = Case(F32, [new] * 5, [max(n, new) for n in (5, 8, 33, 130, 700)], 2, group, dim, 16, device="cuda", starts=False)
    c.q[:, :, 2] = c.q[:, :, 2].abs() + 0.5
    want, tol = c.want()
    for b in range(5):
        at = c.lens[b] - 1
        page, slot = c.table[b, at // c.page].long(), at % c.page
        c.v[page, slot, 1, 3], c.k[page, slot, 0, 2] = bad, bad
    got = c.attend(ctx).double().cpu()
    ctx.sync_check()
    last = torch.zeros(c.tokens, dtype=torch.bool)
    last[[n - 1 for n in c.starts[1:]]] = True
    assert ((got - want).abs() <= tol)[~last].all()
    assert (got[last][:, group:, 3] == bad).all()
    keep = [d for d in range(dim) if d != 3]
    assert ((got - want).abs() <= tol)[last][:, group:][:, :, keep].all()
    if bad > 0:
        assert torch.isnan(got[last][:, :group]).all()  # inf - inf
    else:  # weighs nothing: the same queries without their newest key
        c.lens = [n - 1 for n in c.lens]
        want, tol = c.want(causal=False)
        assert ((got - want).abs() <= tol)[last][:, :group].all()


# ---- more of what the documentation allows --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,lens,prefix", [([2, 0, 3], [60, 9, 700], 0), ([40, 70], [90, 300], 0), ([1, 2, 1], [7, 40, 20], 900), ([30, 60], [30, 300], 900)])
def test_rows_before_the_first_sequence_are_left_alone(ctx, dtype, new, lens, prefix):
    c = Case(dtype, new, lens, 2, 3, 64, 16, prefix=prefix, device="cuda")
    k, v, t, n = arguments(c)
    q, out = (torch.full((c.tokens + 5, 6, 64), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    q[3:-2] = c.on(c.q)
    starts = c.on(c.q_starts) + 3
    if prefix:
        ctx.attention_prefix(q, k, v, c.on(c.prefix_table), prefix, t, n, q_starts=starts, out=out)
    else:
        ctx.attention_paged(q, k, v, t, n, q_starts=starts, out=out)
    c.check(out[3:-2])
    assert (out[:3] == 7).all() and (out[-2:] == 7).all()
    before, out = (k.clone(), v.clone()), torch.full_like(q, 5.0)
    ctx.kv_append(q[:, :2], q[:, 2:4], k, v, t, n, q_starts=starts, q=q, q_out=out)
    ctx.sync_check()
    assert torch.equal(out[3:-2], q[3:-2]) and (out[:3] == 5).all() and (out[-2:] == 5).all()
    changed = sum(min(a, b) for a, b in zip(new, lens))
    assert int(((k != before[0]) & ~(k.isnan() & before[0].isnan())).flatten(2).any(2).sum()) == changed


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 60])
def test_pages_that_several_sequences_share(ctx, dtype, new):
    """Samples of one question: the same pages in several rows of the table, and one page twice in a row."""
    c = Case(dtype, [new] * 4, [200 + b for b in range(4)], 2, 2, 64, 16, device="cuda", garbage=False)
    c.table[1:, :10] = c.table[0, :10]
    c.table[2, 3] = c.table[2, 7]
    c.check(c.attend(ctx))
    ctx.sync_check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group,dim", [(64, 64), (128, 128), (300, 40)])
def test_very_many_query_heads_on_one_key_head(ctx, dtype, group, dim):
    c = Case(dtype, [1, 2, 1], [900, 40, 1], 1, group, dim, 16, device="cuda")
    c.check(c.attend(ctx))
    c = Case(dtype, [1] * 4, [70, 3, 1, 33], 1, group, dim, 16, prefix=300, device="cuda", starts=False)
    c.check(c.attend(ctx))
    ctx.sync_check()


def test_a_first_call_inside_a_capture():
    """A context whose kernels have never run: limits are raised and tensor maps encoded while the stream is captured."""
    from pet_b200.ops import Context
    fresh = Context(0)
    cases = [Case(BF16, [1] * 3, [50, 1, 200], 2, 4, 64, device="cuda", starts=False), Case(F16, [150], [700], 1, 2, 128, device="cuda"),
             Case(F32, [1] * 40, [300] * 40, 2, 2, 128, device="cuda", starts=False), Case(BF16, [1] * 40, [30] * 40, 2, 4, 64, prefix=2000, device="cuda")]
    args = [(c.on(c.q), *arguments(c), c.on(c.q_starts), c.on(c.prefix_table)) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [fresh.attention_prefix(q, k, v, p, c.prefix, t, n, q_starts=s) if c.prefix else fresh.attention_paged(q, k, v, t, n, q_starts=s)
               for c, (q, k, v, t, n, s, p) in zip(cases, args)]
    for _ in range(2):
        graph.replay()
    fresh.sync_check()
    for c, y in zip(cases, got):
        c.check(y)
    del graph
    fresh.close()


def test_workspaces_of_the_library_are_checked(ctx):
    """The C entry points with no workspace, one that is a byte short, one off the grid: refused, and nothing is written."""
    import ctypes as C
    from pet_b200 import lib as L
    lib = L.load()
    for c in (Case(F32, [1] * 40, [3000] * 40, 2, 2, 64, device="cuda", starts=False), Case(BF16, [100], [9000], 1, 1, 64, device="cuda", starts=False),
              Case(BF16, [1] * 40, [30] * 40, 2, 4, 64, prefix=2000, device="cuda", starts=False), Case(BF16, [1] * 3, [30] * 3, 2, 4, 64, prefix=900, device="cuda", starts=False)):
        k, v, t, n = arguments(c)
        q, p = c.on(c.q), c.on(c.prefix_table)
        out = torch.full_like(q, 3.0)
        cache, seqs, *_ = ctx._kv_call(c.tokens, k, v, t, n, None)
        heads, need = q.shape[1], C.c_size_t()
        rows = [L.KV_ROWS.pack(x.data_ptr(), x.stride(0), x.stride(1)) for x in (q, out)]
        assert lib.petb200_attention_paged_workspace(ctx.h, cache, seqs, c.prefix, heads, C.byref(need)) == 0 and need.value > 0
        work = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")

        def run(at, size):
            stream = torch.cuda.current_stream().cuda_stream
            if c.prefix:
                return lib.petb200_attention_prefix_run(ctx.h, cache, seqs, p.data_ptr(), c.prefix, *rows, heads, 1, c.dim ** -0.5, at, size, stream)
            return lib.petb200_attention_paged_run(ctx.h, cache, seqs, *rows, heads, 1, c.dim ** -0.5, at, size, stream)
        for at, size in ((None, 0), (None, need.value), (work.data_ptr(), need.value - 1), (work.data_ptr() + 8, need.value)):
            assert run(at, size) == ERR_INVALID
        ctx.sync_check()
        assert (out == 3).all()
        assert run(work.data_ptr(), need.value) == 0
        c.check(out)
    ctx.sync_check()
