"""GPU parity of attention of new tokens over a paged pool, with and without a sliding window and first tokens, and of its form
for single tokens, against the definition in 64 bits and a bound derived from it (tests/cache_oracle.py)."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests.cache_graph import recorded
from tests.paged_batch import Batch, g
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# What a probability may lose before it meets V: it is rounded once to the type of V (half a step), in fp32 not at all.
PART = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SINGLE = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}   # (of single tokens: in several parts)


def attend(batch, part=None):
    return batch.attend(PART[batch.dtype] if part is None else part)


def check(ops, dev, batch, **more):
    out = torch.full(batch.q.shape, 77.0, dtype=batch.dtype, device=dev)
    got = batch.run(ops, dev, out=out, **more).cpu()
    want, bound, owned = attend(batch)
    oracle.assert_within(got[owned], want[owned], bound[owned])
    assert bool((got[~owned] == 77).all())                          # rows of no sequence are left as they were
    return got


LAYOUTS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (16, 1, 64), (33, 1, 64), (6, 2, 80), (4, 2, 256), (3, 1, 16), (2, 2, 20), (2, 1, 300), (2, 2, 96), (7, 7, 64), (10, 2, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
def test_new_tokens_from_one_to_several_tiles(ops, dev, dtype, heads, kv_heads, d):
    for seed, (new, lens) in enumerate([([1], [1]), ([1, 2, 3], [1, 40, 3]), ([5], [70]), ([33, 1, 20, 64], [33, 65, 150, 64]), ([130, 7], [200, 7]), ([0, 4, 0], [9, 4, 0])]):
        check(ops, dev, Batch(new, lens, heads, kv_heads, d, dtype, 20 + seed, index=torch.int64 if seed % 2 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (65, 70), (200, 0), (31, 1000)])
def test_windows_and_first_tokens(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    for seed, (new, lens) in enumerate([([1, 1, 1], [1, 64, 300]), ([5, 40, 150], [6, 333, 150])]):
        check(ops, dev, Batch(new, lens, heads, kv_heads, d, dtype, 40 + seed, window=window, sinks=sinks, index=torch.int64 if seed % 2 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 2, 128), (6, 1, 80), (2, 1, 256), (1, 1, 20)])
def test_long_sequences_in_few_and_many_shares(ops, dev, dtype, heads, kv_heads, d):
    check(ops, dev, Batch([3, 1], [3000, 17], heads, kv_heads, d, dtype, 60))
    check(ops, dev, Batch([2], [9001], heads, kv_heads, d, dtype, 61))
    check(ops, dev, Batch([40, 1, 1], [2000, 1, 700], heads, kv_heads, d, dtype, 62, window=900, sinks=5))
    check(ops, dev, Batch([70], [1500], heads, kv_heads, d, dtype, 63))


@pytest.mark.parametrize("dtype", TYPES)
def test_more_sequences_than_a_wave_has_lanes(ops, dev, dtype):
    new = [(i * 7) % 5 for i in range(150)]
    check(ops, dev, Batch(new, [n + (i * 13) % 50 for i, n in enumerate(new)], 4, 2, 64, dtype, 70))
    check(ops, dev, Batch([0] * 130 + [3], [5] * 130 + [9], 2, 1, 128, dtype, 71))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 36])
def test_slots_outside_the_pool_and_lengths_outside_the_table(ops, dev, dtype, d):
    b = Batch([20, 9, 4, 6, 5, 3], [60, 200, 4, 33, 7, 40], 4, 2, d, dtype, 80, index=torch.int64, gap=0, tail=4)
    seen = {s for slots in b.slots_of_rows()[0] for s in slots.tolist()}
    swap = next(i for i in range(1, b.k.shape[0]) if i not in seen)
    b.b_loc[b.b_loc == 0] = swap
    b.k[0], b.v[0] = math.nan, math.inf                             # slot 0 stands in for none: whatever is in it must not matter
    at = lambda i, j: (i, b.max_len - b.lens[i] + j)
    b.b_loc[at(0, 10)], b.b_loc[at(0, 59)], b.b_loc[at(0, 0)] = -1, b.k.shape[0], 2 ** 31 + 3
    b.b_loc[1, b.max_len - 200:b.max_len - 100] = -2 ** 33
    b.b_loc[2, b.max_len - 4:b.max_len] = 2 ** 32                   # a sequence with nothing at all: zeros
    got = check(ops, dev, b)
    assert bool((got[b.start[2]:b.start[2] + 4] == 0).all())
    # more new tokens than tokens: those before the first see nothing
    b.tables[2][4] = b.lens[4] = 2
    got = check(ops, dev, b)
    assert bool((got[b.start[4]:b.start[4] + 3] == 0).all())
    b.tables[2][3] = -5                                             # cut to nothing
    b.lens[3] = 0
    check(ops, dev, b)
    b.tables[2][1], b.tables[1][5] = 10 ** 12, -3                   # cut to the table; no new tokens
    b.lens[1], b.new[5] = b.max_len, 0
    check(ops, dev, b)
    b.tables[1][5], b.new[5] = 10 ** 11, b.max_new                  # cut to max_new_len, and to the rows that q has
    b.new[5] = min(b.max_new, b.rows - b.start[5])
    b.lens[5] -= b.max_new - b.new[5]                               # (positions count from the cut length)
    want = b.run(ops, dev, out=torch.full(b.q.shape, 77.0, dtype=dtype, device=dev)).cpu()
    rows = slice(b.start[5], b.start[5] + b.new[5])
    seen = []
    for t in range(b.new[5]):
        p = 40 - b.max_new + t
        seen.append(b.b_loc[5, [b.max_len - 40 + j for j in range(p + 1)]].long())
    full, bound = oracle.attend(b.q[rows], b.k, b.v, seen, PART[dtype])
    oracle.assert_within(want[rows], full, bound + 2.0 ** -20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 20])
def test_rows_outside_q_are_left_out(ops, dev, dtype, d):
    b = Batch([6, 5, 4], [30, 20, 10], 4, 2, d, dtype, 90, gap=0, tail=0, index=torch.int64)
    want = b.run(ops, dev).cpu()
    for start, keep in ((-2, slice(2, 6)), (-100, slice(0, 0)), (13, slice(0, 2)), (2 ** 40, slice(0, 0)), (-2 ** 63, slice(0, 0))):
        b.tables[0][0] = start
        q = b.q.clone()
        if keep.stop > keep.start:
            rows = slice(start + keep.start, start + keep.stop)
            q[rows] = b.q[keep]
        out = torch.full(b.q.shape, 77.0, dtype=dtype, device=dev)
        x = list(b.to(dev))
        x[0] = q.to(dev)
        x[5] = torch.tensor([6, 0, 0], device=dev)
        got = ops.paged_context_attention(*x, out=out).cpu()
        left = torch.ones(b.rows, dtype=torch.bool)
        if keep.stop > keep.start:
            assert_exact(got[rows], want[keep])
            left[rows] = False
        assert bool((got[left] == 77).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (2, 2, 128), (4, 1, 256), (2, 1, 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2), (70, 5)])
def test_what_a_token_does_not_see_does_not_reach_it(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    """Infinities and NaN in the K and V rows of one token: new tokens that see it show them, the others are as exact as ever."""
    b = Batch([40, 3], [150, 90], heads, kv_heads, d, dtype, 95, window=window, sinks=sinks)
    for j in (149, 130, 112, 1) if not window else (149, 130, 1):
        slot = int(b.b_loc[0, b.max_len - 150 + j])
        for rows, value in ((b.k, math.nan), (b.v, math.nan), (b.v, math.inf), (b.v, -math.inf)):
            kept = rows[slot].clone()
            rows[slot, kv_heads - 1, 7] = value
            got = b.run(ops, dev).cpu()
            rows[slot] = kept
            want, bound, owned = attend(b)
            hit = torch.zeros(b.q.shape, dtype=torch.bool)
            for t in range(40):
                if j in b.sees(110 + t):
                    where = hit[b.start[0] + t, heads - heads // kv_heads:]
                    where[:, 7 if rows is b.v else slice(None)] = True
            assert torch.equal(~got[owned].isfinite(), hit[owned])
            assert bool((got[hit].isnan() if math.isnan(value) else got[hit] == value).all())
            ok = owned[:, None, None] & ~hit
            oracle.assert_within(got[ok], want[ok], bound[ok])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(20, 3), (1, 0)])
def test_stale_slots_hold_anything(ops, dev, dtype, window, sinks):
    """Table entries of tokens that have left every window lead to rows of NaN, or outside the pool."""
    b = Batch([30, 1, 2], [300, 200, 100], 4, 2, 64, dtype, 96, window=window, sinks=sinks, index=torch.int64)
    free = next(i for i in range(b.k.shape[0]) if i not in {s for slots in b.slots_of_rows()[0] for s in slots.tolist()})
    b.k[free], b.v[free] = math.nan, math.nan
    for n, length in enumerate(b.lens):
        wanted = set(b.wanted(n))
        for j in range(length):
            if j not in wanted:
                b.b_loc[n, b.max_len - length + j] = free if j % 2 else -7
    check(ops, dev, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [64, 4096, 2.0 ** 40])
def test_scores_of_any_size(ops, dev, dtype, size):
    b = Batch([70, 3], [200, 150], 4, 2, 64, torch.float32, 97)
    top = min(size, 2.0 ** 15) if dtype == torch.float16 else size
    b.q, b.k = torch.sign(b.q) * top, (torch.sign(b.k) * top).to(dtype)
    b.q, b.v, b.dtype = b.q.to(dtype), b.v.to(dtype), dtype
    check(ops, dev, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 36])
def test_small_weights_with_all_of_the_values(ops, dev, dtype, d):
    """One token has nearly all of the weight and no values: what is left of the others counts."""
    b = Batch([33, 2], [400, 300], 2, 2, d, dtype, 98)
    b.q.zero_()
    b.q[..., 0] = math.sqrt(d)
    b.k.zero_()
    b.k[:, :, 0] = torch.rand(b.k.shape[0], 1, generator=g(51)).to(dtype)
    b.v = (1 + torch.rand(b.v.shape, generator=g(52))).to(dtype) * (2.0 ** 12 if dtype != torch.float16 else 2.0 ** 8)
    for n in range(2):
        slot = int(b.b_loc[n, b.max_len - b.lens[n] + 17])
        b.k[slot, :, 0], b.v[slot] = 16, 0
    check(ops, dev, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_scores_and_rows_of_nan_alone(ops, dev, dtype):
    b = Batch([40, 2], [100, 80], 2, 2, 64, dtype, 99)
    row = b.start[0] + 7
    b.q[row, 0] = math.nan                                          # one head of one new token: its row alone
    got = b.run(ops, dev).cpu()
    want, bound, owned = attend(Batch([40, 2], [100, 80], 2, 2, 64, dtype, 99))
    assert bool(got[row, 0].isnan().all())
    owned = owned[:, None].repeat(1, 2)
    owned[row, 0] = False
    oracle.assert_within(got[owned], want[owned], bound[owned])


@pytest.mark.parametrize("dtype", TYPES)
def test_tensors_at_other_strides_and_alignments(ops, dev, dtype):
    for d, shift in [(128, 0), (128, 1), (64, 8), (80, 4), (256, 2)]:
        b = Batch([40, 1, 9], [90, 30, 9], 6, 2, d, dtype, 100, window=50, sinks=2)
        n = b.k.shape[0]
        both = torch.zeros(n * 2 * 2 * (d + 8) + shift, dtype=dtype, device=dev)[shift:].view(n, 2, 2, d + 8)
        both[:, 0, :, :d], both[:, 1, :, :d] = b.k.to(dev), b.v.to(dev)
        rows = torch.randn(b.rows, 10, d, generator=g(71)).to(dtype).to(dev)
        rows[:, 2:8] = b.q.to(dev)
        out = torch.full((b.rows, 8, d + 1), 77.0, dtype=dtype, device=dev)
        wide = torch.zeros(3, b.b_loc.shape[1] + 5, dtype=torch.int32, device=dev)
        wide[:, :b.b_loc.shape[1]] = b.b_loc.to(dev)
        x = b.to(dev)
        ops.paged_context_attention(rows[:, 2:8], both[:, 0, :, :d], both[:, 1, :, :d], wide, *x[4:], window=50, sinks=2, out=out[:, 1:7, :d])
        want, bound, owned = attend(b)
        got = out.cpu()
        oracle.assert_within(got[owned, 1:7, :d], want[owned], bound[owned])
        assert bool((got[~owned] == 77).all() & (got[:, 0] == 77).all() & (got[:, 7] == 77).all() & (got[..., d] == 77).all())


def test_a_pool_past_2_to_the_31_elements(ops, dev):
    slots, heads, d = 270000, 32, 256
    k, v = [torch.zeros(slots, heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    far = torch.tensor([slots - 1, 0, 262150, 131077, slots - 2])
    b = Batch([3, 2], [5, 2], heads, heads, d, torch.bfloat16, 75)
    kk, vv = [torch.randn(5, heads, d, generator=g(s)).bfloat16() for s in (76, 77)]
    k[far.to(dev)], v[far.to(dev)] = kk.to(dev), vv.to(dev)
    b.b_loc[0, :5], b.b_loc[1, 3:5] = far.int(), far[:2].int()
    x = list(b.to(dev))
    got = ops.paged_context_attention(x[0], k, v, *x[3:]).cpu()
    b.k, b.v = kk, vv
    b.b_loc[0, :5] = torch.arange(5).int()
    b.b_loc[1, 3:5] = torch.arange(2).int()
    want, bound, owned = attend(b)
    oracle.assert_within(got[owned], want[owned], bound[owned])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 128), (8, 2, 128), (32, 8, 64), (3, 1, 80), (4, 2, 256), (2, 2, 20), (17, 1, 64), (64, 64, 128), (6, 3, 96), (2, 1, 300)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 3), (100, 0), (100, 4), (600, 5), (40, 100)])
def test_single_tokens(ops, dev, dtype, heads, kv_heads, d, window, sinks):
    """Decode attention with a window; table entries outside it lead to rows of NaN or nowhere."""
    lens = [1, 2, 104, 105, 103, 700, 99, 0, 641, 645]
    new = [1] * len(lens)
    b = Batch(new, [max(n, 1) for n in lens], heads, kv_heads, d, dtype, 110, window=window, sinks=sinks, gap=0, tail=0, index=torch.int64)
    free = next((i for i in range(b.k.shape[0]) if i not in {s for slots in b.slots_of_rows()[0] for s in slots.tolist()}))
    b.k[free], b.v[free] = math.nan, math.nan
    for n, length in enumerate(lens):
        wanted = set(b.wanted(n))
        for j in range(length):
            if j not in wanted:
                b.b_loc[n, b.max_len - length + j] = free if j % 2 else -7
    b.tables[2][7] = b.lens[7] = 0
    q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
    got = ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, window, sinks)
    want, bound, _ = attend(b, SINGLE[dtype])
    oracle.assert_within(got, want, bound)
    assert bool((got[7] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (40, 40)])
def test_single_tokens_of_long_sequences_and_large_batches(ops, dev, dtype, heads, kv_heads):
    for lens, window, sinks in (([5000], 3000, 4), ([5000, 3000], 4999, 1), ([70 + i for i in range(130)], 90, 20), ([300] * 70, 1, 2)):
        if heads == 40:
            lens = lens[:20]
        b = Batch([1] * len(lens), lens, heads, kv_heads, 128, dtype, 115, window=window, sinks=sinks, gap=0, tail=0)
        q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
        got = ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, window, sinks)
        oracle.assert_within(got, *attend(b, SINGLE[dtype])[:2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2)])
def test_infinities_reach_single_tokens_that_see_them(ops, dev, dtype, heads, kv_heads):
    b = Batch([1, 1], [300, 40], heads, kv_heads, 64, dtype, 116, window=50, sinks=3, gap=0, tail=0)
    for j, seen in ((299, True), (250, True), (249, False), (2, True), (3, False)):
        slot = int(b.b_loc[0, j])
        if not seen:
            slot = next(i for i in range(b.k.shape[0]) if i not in {s for slots in b.slots_of_rows()[0] for s in slots.tolist()})
            b.b_loc[0, j] = slot
        for rows, value in ((b.k, math.nan), (b.v, math.nan), (b.v, math.inf), (b.v, -math.inf)):
            kept = rows[slot].clone()
            rows[slot, 1, 7] = value
            q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
            got = ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, 50, 3).cpu()
            rows[slot] = kept
            hit = torch.zeros(b.q.shape, dtype=torch.bool)
            if seen:
                hit[0, heads // 2:, 7 if rows is b.v else slice(None)] = True
            assert torch.equal(~got.isfinite(), hit)
            assert bool((got[hit].isnan() if math.isnan(value) else got[hit] == value).all())
            want, bound, _ = attend(b, SINGLE[dtype])
            oracle.assert_within(got[~hit], want[~hit], bound[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_without_a_window_the_same_as_the_whole_sequence(ops, dev, dtype):
    b = Batch([1] * 5, [1, 900, 33, 64, 200], 8, 2, 128, dtype, 117, gap=0, tail=0)
    q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
    assert_exact(ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, 0, 7), ops.token_decode_attention(q, k, v, loc, start, seq, max_len))
    assert_exact(ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, 2 ** 31 - 1, 2 ** 31 - 1), ops.token_decode_attention(q, k, v, loc, start, seq, max_len))


def test_no_sequences_and_no_tokens(ops, dev):
    k, none, z = torch.ones(4, 2, 64, device=dev), torch.zeros(0, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    assert ops.paged_context_attention(torch.zeros(0, 2, 64, device=dev), k, k, torch.zeros(0, 5, dtype=torch.int32, device=dev), none, none, none, 3, 5).shape == (0, 2, 64)
    out = torch.full((3, 2, 64), 5.0, device=dev)
    loc = torch.zeros(1, 5, dtype=torch.int32, device=dev)
    ops.paged_context_attention(out.clone(), k, k, loc, z, z, z + 5, 0, 5, out=out)
    ops.paged_context_attention(out.clone(), k, k, loc, z, z, z + 5, 7, 5, out=out)
    assert bool((out == 5).all())
    ops.paged_context_attention(out.clone(), k, k, loc[:, :0], z, z + 2, z, 2, 0, out=out)      # new tokens of sequences without any: zeros
    assert bool((out[:2] == 0).all() & (out[2] == 5).all())
    assert ops.token_decode_attention_window(torch.zeros(0, 2, 64, device=dev), k, k, torch.zeros(0, 5, dtype=torch.int32, device=dev), none, none, 5, 3).shape == (0, 2, 64)
    assert bool((ops.token_decode_attention_window(torch.ones(1, 2, 64, device=dev), k, k, loc[:, :0], z, z, 0, 3) == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_that_share_rows_of_q_are_all_walked(ops, dev, dtype):
    """The same table under two sequences that name the same rows: more pieces than rows, and each row has the one result."""
    b = Batch([40, 40, 3], [60, 60, 20], 4, 2, 64, dtype, 118, gap=0, tail=0)
    b.start[1], b.b_loc[1] = b.start[0], b.b_loc[0]
    b.tables[0][1] = b.start[0]
    x = list(b.to(dev))
    x[0] = x[0][torch.cat([torch.arange(40), torch.arange(80, 83)]).to(dev)].contiguous()
    x[4] = torch.tensor([0, 0, 40], dtype=torch.int32, device=dev)
    got = ops.paged_context_attention(*x)
    one = Batch([40, 40, 3], [60, 60, 20], 4, 2, 64, dtype, 118, gap=0, tail=0)
    want = one.run(ops, dev)
    assert_exact(got[:40], want[:40])
    assert_exact(got[40:], want[80:])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_prompt_without_a_cache_as_in_context_attention(ops, dev, dtype):
    b = Batch([150, 64, 7], [150, 64, 7], 8, 2, 128, dtype, 119, gap=0, tail=0)
    rows = torch.cat([b.b_loc[i, b.max_len - n:b.max_len] for i, n in enumerate(b.lens)]).long()
    want, bound, _ = attend(b)
    oracle.assert_within(b.run(ops, dev), want, bound)
    start, _, lens = [t.to(dev) for t in b.tables]
    whole = ops.context_attention(b.q.to(dev), b.k[rows].to(dev), b.v[rows].to(dev), start, lens, 150)
    oracle.assert_within(whole, want, bound + 2.1 * 2.0 ** -25 * 150 * 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 40])
def test_a_prompt_in_pieces_then_single_tokens(ops, dev, dtype, window):
    """A run of the operators together: each step rotates and appends its rows, then attends; all outputs against one pass in 64 bits."""
    heads, kv_heads, d, sinks = 8, 2, 64, 3
    gen, pieces = g(120), [[50, 20], [33, 1], [1, 64], [1, 1], [1, 1]]
    total = [sum(p[i] for p in pieces) for i in range(2)]
    slots = sum(total) + 5
    perm = torch.randperm(slots, generator=gen)
    tokens = [perm[:total[0]], perm[total[0]:sum(total)]]
    rows = [torch.randn(n, heads + 2 * kv_heads, d, generator=gen).to(dtype) for n in total]
    angle = torch.outer(torch.arange(200).double(), 10000.0 ** (-torch.arange(0, d, 2).double() / d))
    cos, sin = angle.cos().float(), angle.sin().float()
    k, v = [torch.zeros(slots, kv_heads, d, dtype=dtype, device=dev) for _ in range(2)]
    outs, rotated, have = [[], []], [[], []], [0, 0]
    for new in pieces:
        x = torch.cat([rows[i][have[i]:have[i] + new[i]] for i in range(2)]).to(dev)
        pos = torch.cat([torch.arange(have[i], have[i] + new[i]) for i in range(2)])
        dest = torch.cat([tokens[i][have[i]:have[i] + new[i]] for i in range(2)])
        q = ops.rotary_dest_index_copy_kv_pair(x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], cos.to(dev), sin.to(dev), dest.to(dev), k, v, positions=pos.to(dev))
        have = [a + n for a, n in zip(have, new)]
        width = max(have)
        loc = torch.zeros(2, width, dtype=torch.int32)
        for i in range(2):
            loc[i, width - have[i]:] = tokens[i][:have[i]].int()
        lens, start = torch.tensor(have, dtype=torch.int32).to(dev), torch.tensor([0, new[0]], dtype=torch.int32).to(dev)
        if new == [1, 1]:
            out = ops.token_decode_attention_window(q, k, v, loc.to(dev), start, lens, width, window, sinks)
        else:
            out = ops.paged_context_attention(q, k, v, loc.to(dev), start, torch.tensor(new, dtype=torch.int32).to(dev), lens, max(new), width, window=window, sinks=sinks)
        for i, part in enumerate(out.cpu().split(new)):
            outs[i].append(part)
        for i, part in enumerate(q.cpu().split(new)):
            rotated[i].append(part)
    for i in range(2):
        b = Batch([total[i]], [total[i]], heads, kv_heads, d, dtype, 1, window=window, sinks=sinks, gap=0, tail=0)
        b.q, b.k, b.v, b.b_loc = torch.cat(rotated[i]), k.cpu(), v.cpu(), tokens[i][None].int()
        half = rows[i][:, heads:heads + kv_heads].double()
        x0, x1, c, s = half[..., :d // 2], half[..., d // 2:], angle[:total[i], None].cos(), angle[:total[i], None].sin()
        want_k = torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1)
        assert bool(((b.k[tokens[i]].double() - want_k).abs() <= oracle.HALF_STEP[dtype] * want_k.abs() + 2.0 ** -21).all())
        assert_exact(b.v[tokens[i]], rows[i][:, heads + kv_heads:])
        want, bound, _ = attend(b)
        oracle.assert_within(torch.cat(outs[i]), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2)])
def test_recorded_into_two_graphs_and_replayed_next_to_eager_calls(ops, dev, pkg, dtype, heads, kv_heads):
    both = [Batch([5, 1, 40], [900, 30, 200], heads, kv_heads, 64, dtype, 130), Batch([3, 2, 1], [2000, 700, 40], heads, kv_heads, 128, dtype, 131, window=300, sinks=4)]
    on = [b.to(dev) for b in both]
    calls = [lambda b=b, x=x: ops.paged_context_attention(*x, window=b.window, sinks=b.sinks) for b, x in zip(both, on)]
    with recorded(ops, pkg, calls[0]) as (first, a), recorded(ops, pkg, calls[1]) as (second, b):
        owned = [x.slots_of_rows()[1] for x in both]
        for i in range(4):
            for x, c in zip(on, both):
                x[0].mul_(0.75)
                x[6].copy_(torch.tensor([c.lens[0] - 100 * i, c.lens[1], c.lens[2] - i]))
            first.replay()
            second.replay()
            first.replay()
            torch.cuda.synchronize()
            kept = a.clone(), b.clone()
            want = calls[0](), calls[1]()
            torch.cuda.synchronize()
            for n in range(2):
                assert_exact(kept[n].cpu()[owned[n]], want[n].cpu()[owned[n]])


@pytest.mark.parametrize("dtype", TYPES)
def test_single_tokens_recorded_into_a_graph(ops, dev, pkg, dtype):
    b = Batch([1, 1, 1], [3000, 700, 40], 8, 2, 128, dtype, 132, window=1500, sinks=4, gap=0, tail=0)
    q, k, v, loc, start, _, seq, _, max_len = b.to(dev)
    call = lambda: ops.token_decode_attention_window(q, k, v, loc, start, seq, max_len, 1500, 4)
    with recorded(ops, pkg, call) as (graph, out):
        for i in range(4):
            q.mul_(0.75)
            seq.copy_(torch.tensor([3000 - 700 * i, 700, 40 - 10 * i]))
            graph.replay()
            torch.cuda.synchronize()
            kept = out.clone()
            want = call()
            torch.cuda.synchronize()
            assert_exact(kept, want)


def test_on_two_streams_at_once(ops, dev):
    both = [Batch([4, 60, 1], [1800, 300, 90], 8, 2, 128, torch.bfloat16, 140 + i) for i in range(2)]
    want = [b.run(ops, dev) for b in both]
    on, streams, got = [b.to(dev) for b in both], [torch.cuda.Stream() for _ in both], [[] for _ in both]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, x in enumerate(on):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_context_attention(*x))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        owned = both[i].slots_of_rows()[1]
        for o in outs:
            assert_exact(o.cpu()[owned], want[i].cpu()[owned])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,heads,kv_heads,d", [(1, 32, 32, 64), (3, 16, 8, 128), (4, 32, 4, 64), (2, 8, 8, 256)])
def test_many_short_sequences(ops, dev, dtype, new, heads, kv_heads, d):
    n = 1100 // kv_heads                                            # more sequences' heads than workgroups run at once
    lens = [new + (17 * b) % (130 if b % 7 else 5) for b in range(n)]
    check(ops, dev, Batch([new] * n, lens, heads, kv_heads, d, dtype, 90))
    check(ops, dev, Batch([min(new, b % 3) for b in range(n)], lens, heads, kv_heads, d, dtype, 91, window=40, sinks=3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_short_pieces_of_many_sequences(ops, dev, dtype, d):
    new = [1 + (11 * b) % 40 for b in range(40)]                    # blocks enough for no shares, of up to seven tiles
    lens = [n + (53 * b) % 400 for b, n in enumerate(new)]
    b = Batch(new, lens, 8, 8, d, dtype, 95)
    b.b_loc[3, :b.max_len - 20] = -1                                # slots outside the pool
    check(ops, dev, b)
    check(ops, dev, Batch(new, lens, 8, 8, d, dtype, 96, window=70, sinks=66, index=torch.int64))
    b = Batch(new, lens, 8, 8, d, dtype, 97)
    b.v[b.b_loc[5, b.max_len - lens[5]].long()] = math.inf          # the first token of one: all of its new ones see it
    got = b.run(ops, dev).cpu()
    rows = slice(b.start[5], b.start[5] + new[5])
    assert bool(torch.isinf(got[rows]).all())
    b.v[b.b_loc[5, b.max_len - lens[5]].long()] = 0
    want, bound, owned = attend(b)
    owned[rows] = False
    oracle.assert_within(got[owned], want[owned], bound[owned])
