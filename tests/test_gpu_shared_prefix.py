"""GPU parity of decode attention with a prefix that all sequences share, against its definition in 64 bits and a bound
derived from it (tests/cache_oracle.py)."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests.cache_graph import recorded
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# what a probability may lose in a product with V: two parts of 8 bits each for 16-bit results, nothing for fp32
PART = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}


def g(seed):
    return torch.Generator().manual_seed(seed)


def batch_of(prefix, lens, heads, kv_heads, d, dtype, seed, index=torch.int32, spare=3):
    """q, the pool, the shared slots and a right-aligned table of own ones; what the table holds elsewhere is foreign."""
    gen = g(seed)
    batch, width, slots = len(lens), max(max(lens), 1) + spare, prefix + sum(max(n, 0) for n in lens) + 7
    q = torch.randn(batch, heads, d, generator=gen).to(dtype)
    k, v = [torch.randn(slots, kv_heads, d, generator=gen).to(dtype) for _ in range(2)]
    b_loc = torch.randint(0, slots, (batch, width), generator=gen).to(index)
    perm, at, max_len = torch.randperm(slots, generator=gen), prefix, width - spare
    for b, n in enumerate(lens):
        n = max(n, 0)
        b_loc[b, max_len - n:max_len] = perm[at:at + n].to(index)
        at += n
    return q, k, v, perm[:prefix].to(index), b_loc, torch.tensor(lens).to(index), max_len


def run(ops, dev, q, k, v, prefix, b_loc, lens, max_len):
    return ops.token_decode_attention_shared_prefix(q.to(dev), k.to(dev), v.to(dev), prefix.to(dev), b_loc.to(dev), torch.zeros_like(lens).to(dev), lens.to(dev), max_len)


def own_and_shared(prefix, b_loc, lens, max_len):
    return [torch.cat([prefix.long(), oracle.slots_of(b_loc, lens, max_len, b)]) for b in range(len(lens))]


def check(ops, dev, q, k, v, prefix, b_loc, lens, max_len):
    got = run(ops, dev, q, k, v, prefix, b_loc, lens, max_len)
    want, bound = oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[q.dtype])
    oracle.assert_within(got, want, bound)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (4, 4, 128), (8, 2, 128), (16, 1, 64), (33, 1, 64), (6, 2, 80), (4, 2, 256), (3, 1, 16), (2, 2, 20), (2, 1, 300), (2, 2, 96)])
def test_prefixes_and_lengths_from_nothing_to_several_shares(ops, dev, dtype, heads, kv_heads, d):
    for seed, (prefix, lens) in enumerate([(1, [1]), (0, [0, 3, 40]), (17, [0, 0]), (16, [5, 0, 33, 1]), (333, [1, 2, 3, 0, 70]), (130, [128, 129, 5] * 7), (64, [1] * 33)]):
        check(ops, dev, *batch_of(prefix, lens, heads, kv_heads, d, dtype, 20 + seed, torch.int64 if seed % 2 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_any_number_of_columns(ops, dev, dtype, d):
    for batch in (8, 9, 12, 13, 17, 20, 21, 25, 29, 33, 37, 41, 49, 53, 57, 65, 69, 97, 101):   # of 4 columns each: 2 to 26 tiles of 16
        check(ops, dev, *batch_of(70 + batch, [batch % 3] * (batch - 1) + [9], 4, 1, d, dtype, 200 + batch))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (1, 1, 128), (4, 4, 80), (6, 2, 128), (5, 1, 256), (7, 1, 72), (18, 1, 64), (3, 3, 96)])
def test_one_to_many_shares_of_the_prefix(ops, dev, dtype, heads, kv_heads, d):
    for prefix in (1, 65, 129, 500, 577, 1000, 2048, 2049, 2113, 4500):   # in shares of 64 or so: up to 32 begin the walk over the own tokens, more are merged
        check(ops, dev, *batch_of(prefix, [3, 0, 20], heads, kv_heads, d, dtype, 300 + prefix))
    check(ops, dev, *batch_of(700, [0, 0], heads, kv_heads, d, dtype, 299, spare=0)[:-1], 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 1, 20), (3, 3, 1), (4, 2, 300), (2, 2, 1024), (1, 1, 513), (8, 2, 256), (2, 1, 132), (2, 1, 250)])
def test_head_sizes_of_any_kind_in_many_chunks(ops, dev, dtype, heads, kv_heads, d):
    for prefix, lens in ((1, [0]), (255, [1, 0]), (256, [0, 700]), (3000, [20, 0, 300]), (5001, [1] * 9)):
        check(ops, dev, *batch_of(prefix, lens, heads, kv_heads, d, dtype, 500 + prefix))
    q, k, v, prefix, b_loc, lens, max_len = batch_of(1500, [500, 3], heads, kv_heads, d, dtype, 499)
    prefix[::3], prefix[512:1024] = -1, k.shape[0] + 5                # some slots, and whole chunks, outside the pool
    got = run(ops, dev, q, k, v, prefix, b_loc, lens, max_len)
    want, bound = oracle.attend(q, k, v, own_and_shared(prefix[(prefix >= 0) & (prefix < k.shape[0])], b_loc, lens, max_len), PART[q.dtype])
    oracle.assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 1)])
def test_shares_without_a_token_that_counts(ops, dev, dtype, heads, kv_heads):
    q, k, v, prefix, b_loc, lens, max_len = batch_of(640, [3, 0, 20], heads, kv_heads, 64, dtype, 310)
    for begin, end in ((0, 64), (64, 200), (0, 640)):                # the first share, one between others, all of them
        some = prefix.clone()
        some[begin:end] = -1
        got = run(ops, dev, q, k, v, some, b_loc, lens, max_len)
        want, bound = oracle.attend(q, k, v, own_and_shared(some[some >= 0], b_loc, lens, max_len), PART[q.dtype])
        oracle.assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_long_prefix_and_long_sequences(ops, dev, dtype):
    check(ops, dev, *batch_of(6001, [1, 700, 30], 4, 2, 128, dtype, 30))
    check(ops, dev, *batch_of(2049, [2600, 1], 2, 2, 64, dtype, 31))
    check(ops, dev, *batch_of(40003, [1], 1, 1, 64, dtype, 32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 36])
def test_slots_outside_the_pool_and_lengths_outside_the_table(ops, dev, dtype, d):
    q, k, v, prefix, b_loc, lens, max_len = batch_of(300, [40, 200, 7, 33, 5], 4, 2, d, dtype, 40, torch.int64)
    slots = k.shape[0]
    seen = set(torch.cat(own_and_shared(prefix, b_loc, lens, max_len)).tolist())
    swap = next(i for i in range(1, slots) if i not in seen)
    b_loc[b_loc == 0] = swap
    prefix[prefix == 0] = swap
    k[0], v[0] = math.nan, math.inf                               # slot 0 stands in for none: whatever is in it must not matter
    prefix[0], prefix[100:140], prefix[299], prefix[250] = -1, slots, -2 ** 40, 2 ** 31 + 1
    b_loc[1, max_len - 200:max_len - 100] = -1
    b_loc[0, max_len - 40] = 2 ** 31 + 3
    b_loc[2, max_len - 7:max_len] = -2 ** 33
    lens[3], lens[4] = -4, 10 ** 6                               # cut to nothing, and to the table
    check(ops, dev, q, k, v, prefix, b_loc, lens, max_len)
    prefix[:] = slots + 1                                         # nothing of the prefix counts; one sequence has nothing at all
    got = check(ops, dev, q, k, v, prefix, b_loc, lens, max_len)
    assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["shared", "own"])
def test_infinities_and_nan_reach_those_that_see_them(ops, dev, dtype, where):
    q, k, v, prefix, b_loc, lens, max_len = batch_of(90, [20, 30, 0], 4, 2, 64, dtype, 45)
    slot = prefix[33] if where == "shared" else b_loc[1, max_len - 5]
    for value, slots_of in [(math.nan, k), (math.nan, v), (math.inf, v), (-math.inf, v)]:
        kept = slots_of[slot].clone()
        slots_of[slot, 1, 7] = value
        got = run(ops, dev, q, k, v, prefix, b_loc, lens, max_len).cpu()
        hit = torch.zeros(3, 4, 64, dtype=torch.bool)
        rows_hit = slice(0, 3) if where == "shared" else slice(1, 2)
        if slots_of is k:
            hit[rows_hit, 2:] = True
        else:
            hit[rows_hit, 2:, 7] = True
        assert torch.equal(~got.isfinite(), hit)
        assert bool((got[hit].isnan() if math.isnan(value) else got[hit] == value).all())
        slots_of[slot] = kept
        want, bound = oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[dtype])
        oracle.assert_within(got[~hit], want[~hit], bound[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_far_apart_between_prefix_and_own_tokens(ops, dev, dtype):
    """One side has all of the weight but no values: what is left of the other counts."""
    heads, d, n = 2, 128, 400
    for top in (17, 390):                                        # among the shared tokens, and among the own ones
        q = torch.zeros(3, heads, d, dtype=dtype)
        q[..., 0] = 1
        k = torch.zeros(n, heads, d, dtype=dtype)
        v = (1 + torch.rand(n, heads, d, generator=g(50))).to(dtype) * (2.0 ** 12 if dtype != torch.float16 else 2.0 ** 8)
        k[:, :, 0] = (torch.rand(n, 1, generator=g(51)) * 30).to(dtype)
        k[top, :, 0], v[top] = 220, 0                             # scores of 0 ... 2.7, and 19.4
        loc = torch.arange(370, 400).repeat(3, 1)
        check(ops, dev, q, k, v, torch.arange(370), loc, torch.tensor([30, 30, 30]), 30)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_the_largest_size(ops, dev, dtype):
    """All of the weight on one key, scores of thousands with either sign."""
    q, k, v, prefix, b_loc, lens, max_len = batch_of(200, [50, 1, 0], 4, 2, 64, torch.float32, 55)
    q = torch.sign(q) * 64
    check(ops, dev, q.to(dtype), (k.sign() * 32).to(dtype), v.to(dtype), prefix, b_loc, lens, max_len)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_numbers_below_the_smallest_normal_one_of_fp16(ops, dev, dtype, d):
    q, k, v, prefix, b_loc, lens, max_len = batch_of(300, [70, 3, 0], 8, 2, d, torch.float32, 65)
    for a, b, c in ((2.0 ** -20, 2.0 ** 13, 1), (2.0 ** 13, 2.0 ** -20, 1), (1, 1, 2.0 ** -18)):
        check(ops, dev, (q * a).to(dtype), (k * b).to(dtype), (v * c).to(dtype), prefix, b_loc, lens, max_len)


@pytest.mark.parametrize("dtype", TYPES)
def test_q_and_pools_at_other_strides_and_alignments(ops, dev, dtype):
    for d, shift in [(128, 0), (128, 1), (64, 8), (80, 4)]:
        q, k, v, prefix, b_loc, lens, max_len = batch_of(150, [33, 0, 200], 6, 2, d, dtype, 70)
        n = k.shape[0]
        both = torch.zeros(n * 2 * 2 * (d + 8) + shift, dtype=dtype, device=dev)[shift:].view(n, 2, 2, d + 8)
        both[:, 0, :, :d], both[:, 1, :, :d] = k.to(dev), v.to(dev)
        rows_q = torch.randn(3, 10, d, generator=g(71)).to(dtype).to(dev)
        rows_q[:, 2:8] = q.to(dev)
        spread = torch.stack([prefix, prefix * 0 - 1], 1).to(dev)[:, 0]
        out = ops.token_decode_attention_shared_prefix(rows_q[:, 2:8], both[:, 0, :, :d], both[:, 1, :, :d], spread, b_loc.to(dev), lens.to(dev), lens.to(dev), max_len)
        oracle.assert_within(out, *oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[dtype]))


def test_a_pool_past_2_to_the_31_elements(ops, dev):
    slots, heads, d = 270000, 32, 256
    k, v = [torch.zeros(slots, heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    far = torch.tensor([slots - 1, 0, 262150, 131077, slots - 2])
    kk, vv = [torch.randn(5, heads, d, generator=g(s)).bfloat16() for s in (75, 76)]
    k[far.to(dev)], v[far.to(dev)] = kk.to(dev), vv.to(dev)
    q = torch.randn(2, heads, d, generator=g(77)).bfloat16()
    loc, lens = far[3:].repeat(2, 1), torch.tensor([2, 1])
    out = run(ops, dev, q, k, v, far[:3], loc, lens, 2)
    oracle.assert_within(out, *oracle.attend(q, kk, vv, [torch.arange(5), torch.tensor([0, 1, 2, 4])], PART[torch.bfloat16]))


def test_the_largest_batch_on_one_head(ops, dev):
    """2.6 million columns: (groups of columns) x (their tiles) pass 2^31."""
    batch, heads, d = 65535, 40, 64
    q, k, v, prefix, b_loc, lens, max_len = batch_of(6, [1] * 2 + [0] + [1] * 3, heads, 1, d, torch.bfloat16, 90)
    at = torch.randint(0, len(lens), (batch,), generator=g(91))
    got = run(ops, dev, q.to(dev)[at.to(dev)], k, v, prefix, b_loc[at], lens[at], max_len)
    want = run(ops, dev, q, k, v, prefix, b_loc, lens, max_len)
    full, bound = oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[q.dtype])
    oracle.assert_within(want, full, bound)
    for first in range(0, batch, 8192):
        some = at[first:first + 8192]
        oracle.assert_within(got[first:first + 8192], full[some], bound[some])


def test_no_sequences(ops, dev):
    k, none = torch.ones(4, 2, 64, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    out = ops.token_decode_attention_shared_prefix(torch.zeros(0, 2, 64, device=dev), k, k, none, torch.zeros(0, 5, dtype=torch.int32, device=dev), none, none, 5)
    assert out.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_as_attention_over_tables_with_the_prefix_written_out(ops, dev, dtype):
    """A batch moves from a table that names the prefix in every row to the shared one: both hold the same bound."""
    q, k, v, prefix, b_loc, lens, max_len = batch_of(500, [20, 1, 90, 300], 8, 2, 128, dtype, 80)
    full = torch.zeros(4, 500 + max_len, dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        full[b, max_len - n:] = torch.cat([prefix, b_loc[b, max_len - n:max_len]])
    whole = ops.token_decode_attention(q.to(dev), k.to(dev), v.to(dev), full.to(dev), lens.to(dev), (lens + 500).to(dev), 500 + max_len)
    want, bound = oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[dtype])
    oracle.assert_within(whole, want, bound)
    oracle.assert_within(run(ops, dev, q, k, v, prefix, b_loc, lens, max_len), want, bound)


def test_decode_steps_behind_a_shared_prefix(ops, dev):
    """New tokens are written into the pool and attended to with the prefix and what each sequence has so far."""
    q, k, v, prefix, b_loc, lens, max_len = batch_of(200, [1, 5, 30], 8, 2, 64, torch.bfloat16, 85, spare=0)
    kd, vd = k.to(dev), v.to(dev)
    for step in range(3):
        new = [torch.randn(3, 2, 64, generator=g(86 + 2 * step + i)).bfloat16() for i in range(2)]
        dest = b_loc[:, -1].contiguous()
        ops.dest_index_copy_kv_pair(new[0].to(dev), new[1].to(dev), dest.to(dev), kd, vd)
        k[dest.long()], v[dest.long()] = new
        got = ops.token_decode_attention_shared_prefix(q.to(dev), kd, vd, prefix.to(dev), b_loc.to(dev), lens.to(dev), lens.to(dev), max_len)
        oracle.assert_within(got, *oracle.attend(q, k, v, own_and_shared(prefix, b_loc, lens, max_len), PART[q.dtype]))
        if step == 2:
            break                                                 # (the pool has no more slots)
        free = torch.tensor([i for i in range(k.shape[0]) if i not in set(torch.cat(own_and_shared(prefix, b_loc, lens, max_len)).tolist())])
        b_loc = torch.cat([b_loc, free[:3, None].to(b_loc.dtype)], 1)
        lens, max_len = lens + 1, max_len + 1


@pytest.mark.parametrize("dtype", TYPES)
def test_recorded_into_a_graph_and_replayed_next_to_eager_calls(ops, dev, pkg, dtype):
    q, k, v, prefix, b_loc, lens, max_len = [t.to(dev) if hasattr(t, "to") else t for t in batch_of(1500, [900, 40, 333], 8, 2, 128, dtype, 100)]
    call = lambda: ops.token_decode_attention_shared_prefix(q, k, v, prefix, b_loc, lens, lens, max_len)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(6):
            before = pkg.runtime.cachingStats()["num_device_malloc"]
            warm = ops.WorkspaceScope()
            with warm:
                call()
            side.synchronize()
            warm.close()
            if pkg.runtime.cachingStats()["num_device_malloc"] == before:
                break
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        scope = ops.WorkspaceScope()
        with scope:
            out = call()
    for i in range(4):
        q.mul_(0.75)
        lens.copy_(torch.tensor([900 - 300 * i, 40, 0 if i else 333]))
        graph.replay()
        torch.cuda.synchronize()
        kept = out.clone()
        want = call()
        torch.cuda.synchronize()
        assert_exact(kept, want)
    del graph
    scope.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1)])
def test_short_sequences_recorded_into_two_graphs(ops, dev, pkg, dtype, heads, kv_heads):
    """The shared tokens' partial results are read by the launch behind, in each graph's own workspace."""
    cases = [[t.to(dev) if hasattr(t, "to") else t for t in batch_of(700 + 300 * i, [20, 3, 11], heads, kv_heads, 64, dtype, 400 + i)] for i in range(2)]
    calls = [lambda c=c: ops.token_decode_attention_shared_prefix(c[0], c[1], c[2], c[3], c[4], c[5], c[5], c[6]) for c in cases]
    with recorded(ops, pkg, calls[0]) as (first, a), recorded(ops, pkg, calls[1]) as (second, b):
        for i in range(4):
            for c in cases:
                c[0].mul_(0.75)
                c[5].copy_(torch.tensor([20 - 5 * i, 3, 0 if i else 11]))
            first.replay()
            second.replay()
            first.replay()
            torch.cuda.synchronize()
            kept = a.clone(), b.clone()
            want = calls[0](), calls[1]()
            torch.cuda.synchronize()
            assert_exact(kept[0], want[0])
            assert_exact(kept[1], want[1])


def test_on_another_stream_with_calls_in_flight_on_the_first(ops, dev):
    cases = [batch_of(1800, [700, 3, 0, 90], 8, 2, 128, torch.bfloat16, 120 + i) for i in range(2)]
    want = [run(ops, dev, *c) for c in cases]
    on = [[t.to(dev) if hasattr(t, "to") else t for t in c] for c in cases]
    streams, got = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (q, k, v, prefix, b_loc, lens, m) in enumerate(on):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.token_decode_attention_shared_prefix(q, k, v, prefix, b_loc, lens, lens, m))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for o in outs:
            assert_exact(o, want[i])
