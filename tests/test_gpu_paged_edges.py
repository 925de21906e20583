"""GPU parity of attention of new tokens over a paged pool where sums are not finite, against the definition in 64 bits
(tests/paged_batch.py)."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests.paged_batch import Batch

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
