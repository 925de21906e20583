"""GPU parity of attention of new tokens over a paged pool, and of decode attention, at their edges (sums and scores that are not finite, workspace, graphs),
against the definition in 64 bits (tests/paged_batch.py, tests/cache_oracle.py)."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests.cache_graph import recorded
from tests.paged_batch import Batch
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# What a probability may lose before it meets V: it is rounded once to the type of V (half a step), in fp32 not at all.
PART = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def damaged(ops, dev, b, n, rows, j, value):
    """Element 7 of the last K/V head's row of token j of sequence n holds `value`: those new tokens that see it show it, all of the others
    are as exact as ever."""
    slot, group = int(b.b_loc[n, b.max_len - b.lens[n] + j]), b.q.shape[1] // b.k.shape[1]
    want, bound, owned = b.attend(PART[b.dtype])
    kept = rows[slot].clone()
    rows[slot, -1, 7] = value
    got = b.run(ops, dev).cpu()
    rows[slot] = kept
    hit = torch.zeros(b.q.shape, dtype=torch.bool)
    for t in range(b.new[n]):
        if j in b.sees(b.lens[n] - b.new[n] + t):
            where = hit[b.start[n] + t, -group:]
            where[:, 7 if rows is b.v else slice(None)] = True
    assert torch.equal(~got[owned].isfinite(), hit[owned])
    assert bool((got[hit].isnan() if math.isnan(value) else got[hit] == value).all())
    ok = owned[:, None, None] & ~hit
    oracle.assert_within(got[ok], want[ok], bound[ok])


# first tokens that reach into the window of the first new token: (window, first tokens, new tokens, all of the sequence's)
OVERLAPS = [(4, 108, 7, 108), (65, 70, 5, 105), (60, 40, 3, 90), (9, 85, 3, 90), (1024, 4, 3, 1027), (600, 300, 5, 700), (2000, 1500, 4, 3000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 2, 128), (4, 4, 80), (2, 1, 256), (2, 1, 20)])
@pytest.mark.parametrize("window,sinks,new,length", OVERLAPS)
def test_rows_that_are_not_finite_where_first_tokens_reach_into_the_window(ops, dev, dtype, heads, kv_heads, d, window, sinks, new, length):
    low = length - new - window + 1                                 # the first token of the first new one's window
    assert 0 < low <= sinks
    for others, lens in (([], []), ([40, 1], [77, 30])):            # few columns alone, and next to blocks of many
        b = Batch([new] + others, [length] + lens, heads, kv_heads, d, dtype, 10 + len(others), window=window, sinks=sinks)
        # the last new token, which the others do not see; a first token, the last of them, one of the window, which all see
        for j, rows, value in ((length - 1, b.k, math.nan), (length - 1, b.v, math.inf), (0, b.v, -math.inf), (sinks - 1, b.v, math.inf), (length - new, b.v, math.nan)):
            damaged(ops, dev, b, 0, rows, j, value)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 64), (16, 8, 80)])
@pytest.mark.parametrize("window,sinks", [(9, 30), (20, 22), (60, 40)])
def test_rows_that_are_not_finite_in_many_short_sequences(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    new = [1 + (5 * b) % 6 for b in range(90)]                      # more heads of sequences than workgroups run at once
    lens = [n + (17 * b) % 90 for b, n in enumerate(new)]
    b = Batch(new, lens, heads, kv_heads, d, dtype, 14, window=window, sinks=sinks)
    reach = [n for n in range(90) if new[n] > 2 and 0 < lens[n] - new[n] - window + 1 <= sinks]
    assert len(reach) > 5
    for n in reach[:3]:
        for j, rows, value in ((lens[n] - 1, b.k, math.nan), (lens[n] - 1, b.v, math.inf), (0, b.v, -math.inf)):
            damaged(ops, dev, b, n, rows, j, value)


def workspace(ops, pkg, call):
    """What the call returns, and the bytes of workspace that it takes."""
    scope = ops.WorkspaceScope()
    with scope:
        before = pkg.runtime.cachingStats()["allocated_bytes"]
        out = call()
        taken = pkg.runtime.cachingStats()["allocated_bytes"] - before
    torch.cuda.synchronize()
    scope.close()
    return out, taken


def wide_table(b, width):
    """The arguments of the batch with a slot table and a longest sequence of `width` tokens."""
    x = list(b.to(torch.device("cuda:0")))
    table = torch.full((len(b.lens), width), -1, dtype=b.b_loc.dtype)
    table[:, width - b.max_len:] = b.b_loc[:, :b.max_len]
    x[3], x[8] = table.to(x[0].device), width
    return x


@pytest.mark.parametrize("dtype,heads,kv_heads,d", [(torch.bfloat16, 32, 8, 128), (torch.float16, 8, 8, 64), (torch.float32, 8, 2, 64)])
def test_partial_results_of_the_new_tokens_that_there_can_be_not_of_all_rows(ops, dev, pkg, dtype, heads, kv_heads, d):
    b = Batch([64], [500], heads, kv_heads, d, dtype, 20, tail=8100)
    out, taken = workspace(ops, pkg, lambda: ops.paged_context_attention(*wide_table(b, 131072)))
    want, bound, owned = b.attend(PART[dtype])
    oracle.assert_within(out.cpu()[owned], want[owned], bound[owned])
    assert 0 < taken <= (2 + d) * 4 * 64 * heads * 64 + (4 << 20)   # (64 new tokens, up to 64 shares)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (2, 2, 128), (6, 1, 80), (2, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 70)])
def test_shares_of_new_tokens_in_a_q_of_many_more_rows(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    b = Batch([70, 50, 0, 66, 1, 3], [1500, 900, 40, 70, 1200, 3], heads, kv_heads, d, dtype, 21, window=window, sinks=sinks, tail=700)
    out = torch.full(b.q.shape, 77.0, dtype=dtype, device=dev)
    got = b.run(ops, dev, out=out).cpu()
    want, bound, owned = b.attend(PART[dtype])
    oracle.assert_within(got[owned], want[owned], bound[owned])
    assert bool((got[~owned] == 77).all())
    for n, j, rows, value in ((0, 1499, b.k, math.nan), (0, 1480, b.v, math.inf), (1, 20, b.v, -math.inf), (4, 1199, b.v, math.inf)):
        damaged(ops, dev, b, n, rows, j, value)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [0, 700])
def test_shares_of_new_tokens_whose_first_rows_lie_before_q(ops, dev, dtype, tail):
    b = Batch([70, 50, 7], [1500, 900, 800], 4, 2, 64, dtype, 22, gap=0, tail=tail)
    want, bound, owned = b.attend(PART[dtype])
    x = list(b.to(dev))
    x[0], x[4] = x[0][9:].contiguous(), x[4] - 9
    out = torch.full(x[0].shape, 77.0, dtype=dtype, device=dev)
    got = ops.paged_context_attention(*x, out=out).cpu()
    oracle.assert_within(got[owned[9:]], want[9:][owned[9:]], bound[9:][owned[9:]])
    assert bool((got[~owned[9:]] == 77).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (8, 8, 64), (10, 2, 80), (4, 4, 256)])
@pytest.mark.parametrize("width", [3100, 16384])
@pytest.mark.parametrize("several", [[1, 3, 2, 1], [1, 40, 3, 1]])
def test_a_batch_with_more_sequences_than_new_tokens(ops, dev, pkg, dtype, heads, kv_heads, d, width, several):
    new, lens = [0] * 300, [5] * 300
    for n, at, length in zip(several, (0, 63, 64, 299), (3000, 1100, 17, 700)):
        new[at], lens[at] = n, max(length, n)
    b = Batch(new, lens, heads, kv_heads, d, dtype, 23, gap=0, tail=2)
    x = wide_table(b, width)
    out = torch.full(b.q.shape, 77.0, dtype=dtype, device=dev)
    got, taken = workspace(ops, pkg, lambda: ops.paged_context_attention(*x, out=out))
    want, bound, owned = b.attend(PART[dtype])
    got = got.cpu()
    oracle.assert_within(got[owned], want[owned], bound[owned])
    assert bool((got[~owned] == 77).all())
    assert 0 < taken <= 2 * (2 + d) * 4 * b.rows * heads * 64 + (4 << 20)   # (up to 64 shares of each row, for few columns and for many)
    for n, j, value in ((0, 2999, math.inf), (0, 1500, math.nan), (299, 3, -math.inf)):
        damaged(ops, dev, b, n, b.v, j, value)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 128), (32, 8, 128), (40, 40, 64)])
def test_workspace_of_few_new_tokens_is_that_of_their_columns(ops, dev, pkg, dtype, heads, kv_heads, d):
    b = Batch([1, 1], [900, 300], heads, kv_heads, d, dtype, 24, gap=0, tail=0)
    x = wide_table(b, 32768)
    got, taken = workspace(ops, pkg, lambda: ops.paged_context_attention(*x))
    want, bound, owned = b.attend(PART[dtype])
    oracle.assert_within(got.cpu()[owned], want[owned], bound[owned])
    assert 0 < taken <= (2 + d) * 4 * 2 * heads * 64 + 4096


FORMS = [(8, 2, 64), (4, 4, 128), (6, 1, 80), (2, 1, 256), (2, 1, 20)]


def scored(seed, new, lens, heads, kv_heads, d, dtype, **more):
    """A batch whose q has ones as its element 3: an infinity there in a row of K is that token's score."""
    b = Batch(new, lens, heads, kv_heads, d, dtype, seed, **more)
    b.q[..., 3] = 1
    return b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", FORMS)
def test_infinite_scores_of_single_tokens_with_a_window(ops, dev, dtype, heads, kv_heads, d):
    """As in attention of several new tokens, and as in decode attention without a window."""
    group = heads // kv_heads
    for window, sinks in ((0, 0), (50, 4)):
        b = scored(33, [1, 1, 1], [300, 80, 40], heads, kv_heads, d, dtype, window=window, sinks=sinks, gap=0, tail=0)
        slots = [[int(b.b_loc[n, b.max_len - b.lens[n] + j]) for j in b.wanted(n)] for n in range(3)]
        b.k[slots[0], -1, 3] = -math.inf
        b.k[slots[1][::2], -1, 3] = -math.inf
        b.k[slots[2][3], -1, 3] = math.inf
        q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
        got = ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, window, sinks).cpu()
        assert bool((got[0, -group:] == 0).all() & got[2, -group:].isnan().all())
        b.k[slots[0] + slots[2], -1, 3] = 0
        b.k[slots[1][::2], -1, 3] = 0
        for j in b.wanted(1)[::2]:
            b.b_loc[1, b.max_len - 80 + j] = -1
        want, bound, _ = b.attend(2.0 ** -16 if dtype != torch.float32 else PART[dtype])
        oracle.assert_within(got[1, -group:], want[1, -group:], bound[1, -group:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 96, 112, 20, 24, 160, 256])
@pytest.mark.parametrize("batch,length,kv_heads", [(3, 900, 2), (64, 40, 8), (300, 20, 8)])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_scores_of_minus_infinity_in_decode_attention(ops, dev, dtype, d, batch, length, kv_heads, group):
    """A key with an infinity that makes its score minus infinity weighs nothing, with heads of any size and whichever pipe takes them; alone and behind
    a shared prefix."""
    b = scored(34, [1] * batch, [length - n % 7 for n in range(batch)], group * kv_heads, kv_heads, d, dtype, gap=0, tail=0)
    slots = [[int(b.b_loc[n, b.max_len - b.lens[n] + j]) for j in range(b.lens[n])] for n in range(batch)]
    table, keys = b.b_loc.clone(), b.k.clone()
    for n in range(0, batch, 5):
        at = range(0, b.lens[n], 3)
        keys[[slots[n][j] for j in at], :, 3] = -math.inf
        b.b_loc[n, [b.max_len - b.lens[n] + j for j in at]] = -1
    part = 2.0 ** -16 if dtype != torch.float32 else PART[dtype]
    want, bound, _ = b.attend(part)
    rest, b.b_loc = b.b_loc, table
    q, _, v, loc, start, _, seq, _, max_len = b.to(dev)
    oracle.assert_within(ops.token_decode_attention(q, keys.to(dev), v, loc, start, seq, max_len), want, bound)
    prefix = torch.tensor(slots[1], device=dev)
    got = ops.token_decode_attention_shared_prefix(q, keys.to(dev), v, prefix, loc, start, seq, max_len)
    seen = [torch.cat([torch.tensor(slots[1]), rest[n, b.max_len - b.lens[n]:b.max_len].long()]) for n in range(batch)]
    some = [0, 1, 2, 5, batch - 1] if batch > 3 else [0, 1, 2]
    want, bound = oracle.attend(b.q[some], b.k, b.v, [seen[n] for n in some], part)
    oracle.assert_within(got[some], want, bound)
def with_scores(ops, dev, b, low, high=()):
    """The last K/V head's scores of tokens `low` ((sequence, token) pairs) are minus infinity, those of `high` infinity: the first weigh nothing, as
    tokens that are skipped; new tokens that see one of the others give NaN, whose weight is infinity / infinity."""
    slot = lambda n, j: int(b.b_loc[n, b.max_len - b.lens[n] + j])
    group, kept, table = b.q.shape[1] // b.k.shape[1], b.k.clone(), b.b_loc.clone()
    want, bound, owned = b.attend(PART[b.dtype])
    for n, j in low:
        b.b_loc[n, b.max_len - b.lens[n] + j] = -1
    last, last_bound, _ = b.attend(PART[b.dtype])
    b.b_loc = table
    want[:, -group:], bound[:, -group:] = last[:, -group:], last_bound[:, -group:]
    for pairs, value in ((low, -math.inf), (high, math.inf)):
        for n, j in pairs:
            b.k[slot(n, j), -1, 3] = value
    got = b.run(ops, dev).cpu()
    b.k = kept
    nan = torch.zeros(b.q.shape, dtype=torch.bool)
    for n, j in high:
        for t in range(b.new[n]):
            if j in b.sees(b.lens[n] - b.new[n] + t):
                nan[b.start[n] + t, -group:] = True
    assert torch.equal(got[owned].isnan(), nan[owned])
    ok = owned[:, None, None] & ~nan
    oracle.assert_within(got[ok], want[ok], bound[ok])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", FORMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 60), (90, 4)])
def test_scores_that_are_infinite(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    for new, lens in (([40, 3, 1], [150, 90, 70]), ([3, 1], [90, 70])):         # blocks and few columns, few columns alone
        b = scored(30, new, lens, heads, kv_heads, d, dtype, window=window, sinks=sinks)
        seen = [b.wanted(n) for n in range(len(new))]
        some = [(n, j) for n in range(len(new)) for j in seen[n][::3]]
        with_scores(ops, dev, b, some)
        with_scores(ops, dev, b, [(n, j) for n in range(len(new)) for j in seen[n][:-2]])                      # all that come before the last two
        with_scores(ops, dev, b, some, [(0, lens[0] - 1), (1, lens[1] - new[1])])
        with_scores(ops, dev, b, [], [(0, seen[0][0]), (1, seen[1][-1])])
        got = with_scores(ops, dev, b, [(n, j) for n in range(len(new)) for j in seen[n]])                     # no others: zeros, as without tokens
        owned = b.slots_of_rows()[1]
        assert bool((got[owned][:, -(heads // kv_heads):] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", FORMS)
@pytest.mark.parametrize("new,tail", [(70, 0), (70, 500), (3, 0)])
def test_scores_that_are_infinite_in_some_of_the_shares(ops, dev, dtype, heads, kv_heads, d, new, tail):
    b = scored(31, [new], [2600], heads, kv_heads, d, dtype, tail=tail)
    with_scores(ops, dev, b, [(0, j) for j in range(1300)])                                                    # the first shares altogether
    with_scores(ops, dev, b, [(0, j) for j in range(700, 2600 - new)])
    with_scores(ops, dev, b, [(0, j) for j in range(1300)], [(0, 2000)])
    with_scores(ops, dev, b, [(0, j) for j in range(2600) if j != 5])
    got = with_scores(ops, dev, b, [(0, j) for j in range(2600)])
    assert bool((got[b.start[0]:b.start[0] + new, -(heads // kv_heads):] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", FORMS)
def test_an_infinity_in_q(ops, dev, dtype, heads, kv_heads, d):
    """Scores of a head of one new token are infinities of K's signs: NaN where one is positive, zeros where all are negative, the other rows as ever."""
    for new, lens in (([40, 3], [150, 90]), ([3], [2000])):
        b = scored(32, new, lens, heads, kv_heads, d, dtype)
        n = len(new) - 1
        b.k[..., 3] = -b.k[..., 3].abs() - 0.5
        b.k[int(b.b_loc[n, b.max_len - lens[n] + lens[n] - 2]), -1, 3] = 2       # the last but one of the last sequence
        want, bound, owned = b.attend(PART[dtype])
        first, last = b.start[n], b.start[n] + new[n] - 1
        b.q[first, -1, 3] = b.q[last, -1, 3] = math.inf
        got = b.run(ops, dev).cpu()
        assert bool((got[first, -1] == 0).all() & got[last, -1].isnan().all())
        owned = owned[:, None].repeat(1, heads)
        owned[first, -1] = owned[last, -1] = False
        oracle.assert_within(got[owned], want[owned], bound[owned])




@pytest.mark.parametrize("dtype", TYPES)
def test_calls_with_room_for_more_rows_or_sequences_recorded_into_graphs(ops, dev, pkg, dtype):
    """A q of many more rows than new tokens, and a batch with more sequences than rows, whose tables change between the replays."""
    padded = Batch([66, 3, 5], [1200, 900, 40], 8, 2, 64, dtype, 40, tail=900)
    sparse = Batch([0] * 50 + [2, 0, 1], [7] * 50 + [1500, 9, 800], 8, 2, 64, dtype, 41, gap=0, tail=0)
    on = [b.to(dev) for b in (padded, sparse)]
    outs = [torch.full(b.q.shape, 77.0, dtype=dtype, device=dev) for b in (padded, sparse)]
    calls = [lambda x=x, out=out: ops.paged_context_attention(*x, out=out) for x, out in zip(on, outs)]
    owned = [b.slots_of_rows()[1] for b in (padded, sparse)]
    with recorded(ops, pkg, calls[0]) as (first, _), recorded(ops, pkg, calls[1]) as (second, _):
        for i in range(4):
            for x, b in zip(on, (padded, sparse)):
                x[0].mul_(0.75)
                x[6].copy_(torch.tensor([max(b.new[n], length - 60 * i) for n, length in enumerate(b.lens)]))
            for out in outs:
                out.fill_(77)
            first.replay()
            second.replay()
            first.replay()
            torch.cuda.synchronize()
            kept = [out.cpu() for out in outs]
            for call in calls:
                call()
            torch.cuda.synchronize()
            for got, out, rows in zip(kept, outs, owned):
                assert_exact(got[rows], out.cpu()[rows])
                assert bool((got[~rows] == 77).all())
