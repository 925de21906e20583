"""GPU parity of the int8 KV cache: rows quantised as they are written, read back, and attended to, against definitions in
64 bits (tests/cache_oracle.py). Writing and reading are exact; attention's tolerance is derived there."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests.cache_graph import recorded
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# what a probability may lose in a product: two parts of 8 bits each for 16-bit results, three for fp32
PART = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -24}


def g(seed):
    return torch.Generator().manual_seed(seed)


def rows(tokens, heads, d, dtype, seed):
    """Normal numbers, the heads of different sizes."""
    x = torch.randn(tokens, heads, d, generator=g(seed)) * torch.logspace(-2, 2, heads)[:, None]
    return x.to(dtype)


def empty_pools(slots, heads, d, seed=99):
    """Two pools with something in them already, to see what is left alone."""
    gen = g(seed)
    return [(torch.randint(-127, 128, (slots, heads, d), generator=gen, dtype=torch.int8), torch.rand(slots, heads, generator=gen)) for _ in range(2)]


def check_write(ops, dev, k, v, dest, slots, kd=None, vd=None):
    (kp, ks), (vp, vs) = empty_pools(slots, k.shape[1], k.shape[2])
    got = [t.to(dev) for t in (kp, ks, vp, vs)]
    kd, vd = k.to(dev) if kd is None else kd, v.to(dev) if vd is None else vd
    ops.dest_index_copy_kv_pair_int8(kd, vd, dest.to(dev), *got)
    for have, want in zip(got, oracle.write(kp, ks, k, dest) + oracle.write(vp, vs, v, dest)):
        same = (have.cpu() == want) | (have.cpu().isnan() & want.isnan()) if want.is_floating_point() else have.cpu() == want
        assert bool(same.all()), f"{int((~same).sum())} of {want.numel()} differ"


# ------------------------------------------------------------------ writing
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,d", [(1, 1, 64), (1, 8, 128), (7, 3, 80), (64, 32, 128), (5, 2, 256), (33, 5, 8), (3, 1, 1), (9, 2, 20),
                                            (4, 3, 300), (1500, 4, 96), (2050, 1, 64), (9000, 2, 16)])
def test_rows_are_quantised_to_the_nearest(ops, dev, dtype, tokens, heads, d):
    slots = tokens + 11
    dest = torch.randperm(slots, generator=g(1))[:tokens].to(torch.int32 if tokens % 2 else torch.int64)
    check_write(ops, dev, rows(tokens, heads, d, dtype, 2), rows(tokens, heads, d, dtype, 3), dest, slots)


def test_halves_go_to_the_even_neighbour(ops, dev):
    row = torch.tensor([127., .5, 1.5, 2.5, 3.5, -.5, -1.5, -2.5, 126.5, 125.5, -126.5, 63.5, 64.5, .25, -.75, 0.])
    k = torch.stack([row * 2.0 ** e for e in (-140, -126, -70, -30, 0, 5, 100, 120)])[:, None, :]     # down to scales of few bits
    assert (k[4, 0, 1:8] == row[1:8]).all()
    check_write(ops, dev, k, -k, torch.arange(8), 9)


@pytest.mark.parametrize("dtype", TYPES)
def test_quotients_next_to_a_half(ops, dev, dtype):
    """Rows whose elements are the numbers of the type around (n + 1/2) s, for every n."""
    most = torch.tensor([1.0, 1.37, 100.0, 3.0e-3]).to(dtype)
    s = (most.double() / 127).float().double()
    x = ((torch.arange(-127, 127).double() + 0.5)[None, :, None] * s[:, None, None])
    x = torch.cat([x.to(dtype), (x * (1 + 2.0 ** -10)).to(dtype), (x * (1 - 2.0 ** -10)).to(dtype)], -1).view(4, -1)
    x = torch.cat([x.clamp(-most[:, None], most[:, None]), most[:, None].expand(4, 6)], -1)           # 768 elements
    k = x.view(4, 6, 128).clone()
    k[:, :, 0] = most[:, None]
    check_write(ops, dev, k, -k, torch.tensor([3, 0, 2, 1]), 4)


def test_rows_of_zeros_infinities_nan_and_the_smallest_and_largest_numbers(ops, dev):
    for dtype in TYPES:
        top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        k = rows(8, 2, 64, dtype, 5)
        k[0] = 0
        k[1, 0, 3], k[1, 1, 63] = math.inf, -math.inf
        k[2, 0, 0] = math.nan
        k[3, 1] = top
        k[4] = k[4] * 0 + tiny
        k[5, 0], k[5, 0, 7] = 0, tiny * torch.finfo(dtype).eps                                         # the smallest number there is
        k[6, 0], k[6, 0, :3] = 0, torch.tensor([5, -3, 1]) * tiny * torch.finfo(dtype).eps
        k[7, 1, 5] = -top
        check_write(ops, dev, k, k.flip(0), torch.arange(8), 8)
        check_write(ops, dev, k[..., :50].contiguous(), k[..., 14:].contiguous()[..., :50], torch.arange(8), 8)


@pytest.mark.parametrize("tokens", [6, 1100, 16384, 16385, 20001])
def test_negative_foreign_and_repeated_destinations(ops, dev, tokens):
    slots = 5 + tokens // 3                                      # every slot is named several times
    dest = torch.randint(-slots - 4, slots + 4, (tokens,), generator=g(tokens))
    dest[0], dest[1], dest[-1] = slots - 1, -1, -1 if tokens % 2 else 2 ** 40
    check_write(ops, dev, rows(tokens, 2, 24, torch.bfloat16, 6), rows(tokens, 2, 24, torch.bfloat16, 7), dest, slots)
    same = torch.full((tokens,), 3, dtype=torch.int32)
    check_write(ops, dev, rows(tokens, 1, 20, torch.float16, 8), rows(tokens, 1, 20, torch.float16, 9), same, slots)


@pytest.mark.parametrize("tokens", [4096, 4097])
def test_repeats_where_they_begin_to_be_found_beforehand(ops, dev, tokens):
    dest = torch.randint(0, tokens // 2, (tokens,), generator=g(tokens))
    check_write(ops, dev, rows(tokens, 8, 64, torch.bfloat16, 6), rows(tokens, 8, 64, torch.bfloat16, 7), dest, tokens // 2 + 9)
    check_write(ops, dev, rows(tokens, 1, 128, torch.float32, 6), rows(tokens, 1, 128, torch.float32, 7), dest - tokens // 2, tokens // 2)


@pytest.mark.parametrize("apart", [2 ** 24 - 8, 2 ** 24])        # tokens just below and at the widest step of the kernel with 24-bit products
def test_tokens_far_apart(ops, dev, apart):
    on = torch.empty(2 * apart + 512, dtype=torch.bfloat16, device=dev).as_strided((3, 4, 128), (apart, 128, 1))
    k = rows(3, 4, 128, torch.bfloat16, 15)
    on.copy_(k)
    check_write(ops, dev, k, k, torch.tensor([4, 0, 2]), 5, on, on)
    (kp, ks), (vp, vs) = empty_pools(5, 4, 128)
    index = torch.tensor([4, 1, 3])
    out = torch.empty(2, 2 * apart + 512, dtype=torch.bfloat16, device=dev).as_strided((2, 3, 4, 128), (2 * apart + 512, apart, 128, 1))
    ops.index_select_kv_pair_int8(kp.to(dev), ks.to(dev), vp.to(dev), vs.to(dev), index.to(dev), out_k=out[0], out_v=out[1])
    assert_exact(out.contiguous(), torch.stack([oracle.read(kp, ks, index, torch.bfloat16), oracle.read(vp, vs, index, torch.bfloat16)]))


def test_rows_and_pools_at_other_strides(ops, dev):
    for d, shift in [(128, 0), (64, 3), (40, 8)]:                # whole vectors, a base that is not aligned, half a vector aside
        stacked = torch.randn(21, 6, d, generator=g(10)).bfloat16()
        on = torch.zeros(21 * 6 * d + shift, dtype=torch.bfloat16, device=dev)[shift:].view(21, 6, d).copy_(stacked)
        check_write(ops, dev, stacked[:, 2:4], stacked[:, 4:], torch.arange(21) * 2, 43, on[:, 2:4], on[:, 4:])
        k, v = stacked[:, :2], stacked[:, 3:5]
        both = torch.zeros(30, 2, 2, d + 8, dtype=torch.int8, device=dev)                            # K and V of a slot side by side
        scales = torch.full((2, 2, 30), 7.0, device=dev)
        kp, vp, ks, vs = both[:, 0, :, :d], both[:, 1, :, :d], scales[0].t(), scales[1].t()
        dest = torch.randperm(30, generator=g(11))[:21]
        ops.dest_index_copy_kv_pair_int8(k.to(dev).transpose(0, 1).contiguous().transpose(0, 1), v.to(dev), dest.to(dev), kp, ks, vp, vs)
        wk, wks = oracle.write(torch.zeros(30, 2, d, dtype=torch.int8), torch.full((30, 2), 7.0), k, dest)
        wv, wvs = oracle.write(torch.zeros(30, 2, d, dtype=torch.int8), torch.full((30, 2), 7.0), v, dest)
        assert_exact(both[..., :d].transpose(1, 0).contiguous(), torch.stack([wk, wv]))
        assert int(both[..., d:].abs().max()) == 0
        assert_exact(scales.contiguous(), torch.stack([wks.t(), wvs.t()]))
        for dtype in TYPES:
            out = torch.full((2, 21, 2, d + 8), 5.0, dtype=dtype, device=dev)
            ops.index_select_kv_pair_int8(kp, ks, vp, vs, dest.to(dev), out_k=out[0, ..., :d], out_v=out[1, ..., :d])
            assert_exact(out[..., :d].contiguous(), torch.stack([oracle.read(wk, wks, dest, dtype), oracle.read(wv, wvs, dest, dtype)]))
            assert bool((out[..., d:] == 5).all())


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,d", [(0, 2, 64), (1, 1, 64), (5, 8, 128), (300, 3, 80), (2100, 2, 256), (9, 2, 8), (7, 3, 20), (3, 1, 300), (9000, 1, 16)])
def test_rows_are_read_back(ops, dev, dtype, n, heads, d):
    (kp, ks), (vp, vs) = empty_pools(n // 2 + 5, heads, d)
    ks[1], vs[2] = math.nan, 0
    index = torch.randint(-3, kp.shape[0] + 3, (n,), generator=g(12)).to(torch.int64 if n % 2 else torch.int32)   # repeated, and some outside
    if n > 3:
        index[0], index[1], index[2] = 1, 2, -2 ** 31
    got = ops.index_select_kv_pair_int8(kp.to(dev), ks.to(dev), vp.to(dev), vs.to(dev), index.to(dev), dtype=dtype)
    for have, want in zip(got, (oracle.read(kp, ks, index, dtype), oracle.read(vp, vs, index, dtype))):
        assert have.dtype == dtype and have.shape == (n, heads, d)
        assert torch.equal(have.cpu().nan_to_num(123.0), want.nan_to_num(123.0))


def test_strided_index_and_a_pool_past_2_to_the_31_elements(ops, dev):
    slots, heads, d = 270000, 32, 256                            # 2.2e9 elements a pool
    kp = torch.zeros(slots, heads, d, dtype=torch.int8, device=dev)
    vp, ks, vs = torch.zeros_like(kp), torch.zeros(slots, heads, device=dev), torch.zeros(slots, heads, device=dev)
    k, v = rows(4, heads, d, torch.bfloat16, 13), rows(4, heads, d, torch.bfloat16, 14)
    dest = torch.tensor([slots - 1, 0, 262150, 131077])
    spread = torch.stack([dest, torch.full_like(dest, 5)], 1).to(dev)[:, 0]
    ops.dest_index_copy_kv_pair_int8(k.to(dev), v.to(dev), spread, kp, ks, vp, vs)
    got = ops.index_select_kv_pair_int8(kp, ks, vp, vs, spread, dtype=torch.float32)
    for have, x in zip(got, (k, v)):
        q, s = oracle.quantise(x)
        assert_exact(have, q.float() * s[..., None])
    loc = dest.view(1, 4).to(dev)
    q = torch.randn(1, heads, d, generator=g(15)).bfloat16()
    out = ops.token_decode_attention_int8(q.to(dev), kp, ks, vp, vs, loc, torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 4, device=dev), 4)
    want, bound = oracle.attend(q, got[0].cpu().double(), got[1].cpu().double(), [torch.arange(4)], PART[torch.bfloat16])
    oracle.assert_within(out, want, bound)


# ------------------------------------------------------------------ attention
def batch_of(lens, heads, kv_heads, d, dtype, seed, index=torch.int32, spare=3):
    """q, an int8 pool and a right-aligned table for sequences of these lengths; what the table holds elsewhere is foreign."""
    gen = g(seed)
    batch, width, slots = len(lens), max(max(lens), 1) + spare, sum(max(n, 0) for n in lens) + 7
    q = torch.randn(batch, heads, d, generator=gen).to(dtype)
    pools = [(torch.randint(-127, 128, (slots, kv_heads, d), generator=gen, dtype=torch.int8), (0.2 + torch.rand(slots, kv_heads, generator=gen)) / 40) for _ in range(2)]
    b_loc = torch.randint(0, slots, (batch, width), generator=gen).to(index)
    perm, at, max_len = torch.randperm(slots, generator=gen), 0, width - spare
    for b, n in enumerate(lens):
        n = max(n, 0)
        b_loc[b, max_len - n:max_len] = perm[at:at + n].to(index)
        at += n
    return q, pools, b_loc, torch.tensor(lens).to(index), max_len


def run_attention(ops, dev, q, pools, b_loc, lens, max_len):
    (kp, ks), (vp, vs) = pools
    return ops.token_decode_attention_int8(q.to(dev), kp.to(dev), ks.to(dev), vp.to(dev), vs.to(dev), b_loc.to(dev), torch.zeros_like(lens).to(dev), lens.to(dev), max_len)


def check_attention(ops, dev, q, pools, b_loc, lens, max_len):
    (kp, ks), (vp, vs) = pools
    got = run_attention(ops, dev, q, pools, b_loc, lens, max_len)
    slots = [oracle.slots_of(b_loc, lens, max_len, b) for b in range(len(lens))]
    want, bound = oracle.attend(q, kp.double() * ks.double()[..., None], vp.double() * vs.double()[..., None], slots, PART[q.dtype])
    oracle.assert_within(got, want, bound)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (4, 4, 128), (8, 2, 128), (8, 1, 64), (32, 1, 128), (17, 1, 64), (6, 2, 80), (4, 2, 256), (3, 1, 16), (4, 4, 20),
                                              (2, 1, 300), (2, 2, 112), (1, 1, 1)])
def test_attention_over_lengths_from_nothing_to_several_shares(ops, dev, dtype, heads, kv_heads, d):
    for seed, lens in enumerate([[1], [0, 1, 2], [31, 32, 33, 15, 16, 17], [700, 3, 0, 129], [64, 63, 65, 1, 127, 128, 5, 300]]):
        check_attention(ops, dev, *batch_of(lens, heads, kv_heads, d, dtype, 20 + seed, torch.int64 if seed % 2 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_over_a_long_sequence(ops, dev, dtype):
    check_attention(ops, dev, *batch_of([5000], 4, 2, 128, dtype, 30))
    check_attention(ops, dev, *batch_of([20011, 100], 2, 2, 64, dtype, 31))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 36])
def test_slots_outside_the_pool_and_lengths_outside_the_table(ops, dev, dtype, d):
    q, pools, b_loc, lens, max_len = batch_of([40, 200, 7, 33, 5], 4, 2, d, dtype, 40, torch.int64)
    slots = pools[0][0].shape[0]
    used = torch.cat([oracle.slots_of(b_loc, lens, max_len, b) for b in range(5)])
    for pool, scale in pools:                                     # slot 0 stands in for none: whatever is in it must not matter
        swap = [i for i in range(1, slots) if i not in used.tolist()][0]
        b_loc[b_loc == 0] = swap
        pool[0], scale[0] = 127, math.nan
    b_loc[1, max_len - 200:max_len - 100] = -1
    b_loc[1, max_len - 50:max_len:3] = slots + 5
    b_loc[0, max_len - 40] = 2 ** 31 + 3
    b_loc[2, max_len - 7:max_len] = -2 ** 33                     # nothing is left of this one
    lens[3], lens[4] = -4, 10 ** 6                               # cut to nothing, and to the table
    got = check_attention(ops, dev, q, pools, b_loc, lens, max_len)
    assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 1, 20), (3, 3, 1), (4, 2, 300), (2, 2, 1024), (8, 2, 100), (2, 1, 250)])
def test_head_sizes_of_any_kind_in_many_chunks(ops, dev, dtype, heads, kv_heads, d):
    for seed, lens in enumerate(([0], [1, 0, 255], [256, 257], [20, 0, 3300], [64] * 9)):
        check_attention(ops, dev, *batch_of(lens, heads, kv_heads, d, dtype, 200 + seed, torch.int64 if seed % 2 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_far_above_the_rest_and_values_only_below_it(ops, dev, dtype):
    """The key with almost all of the weight has V = 0: what is left of each of the others counts."""
    heads, d, n = 2, 128, 400
    q = torch.zeros(1, heads, d, dtype=dtype)
    q[..., 0] = 1
    kp, vp = torch.zeros(n, heads, d, dtype=torch.int8), torch.randint(1, 128, (n, heads, d), generator=g(50), dtype=torch.int8)
    kp[:, :, 0] = torch.randint(0, 20, (n, 1), generator=g(51)).to(torch.int8)
    kp[17, :, 0], vp[17] = 127, 0
    ks, vs = torch.full((n, heads), 1.6), torch.full((n, heads), 2.0 ** 12 if dtype != torch.float16 else 2.0 ** 8)   # scores of 0 ... 2.7, and 18
    loc = torch.randperm(n, generator=g(52))[None]
    check_attention(ops, dev, q, [(kp, ks), (vp, vs)], loc, torch.tensor([n]), n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 20])
def test_q_below_the_smallest_normal_number_of_fp16(ops, dev, dtype, d):
    q, pools, b_loc, lens, max_len = batch_of([70, 3, 150], 4, 2, d, dtype, 65)
    (kp, ks), (vp, vs) = pools
    q, ks = (q.float() * 2.0 ** -20).to(dtype), ks * 2.0 ** 20      # scores as they were
    check_attention(ops, dev, q, [(kp, ks), (vp, vs)], b_loc, lens, max_len)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 20])
def test_scales_that_are_nan_infinite_huge_and_zero(ops, dev, dtype, d):
    q, pools, b_loc, lens, max_len = batch_of([70, 70, 70, 70, 90], 2, 1, d, dtype, 60, torch.int64)
    (kp, ks), (vp, vs) = pools
    own = [oracle.slots_of(b_loc, lens, max_len, b) for b in range(5)]
    ks[own[0][5]] = math.nan                                      # a row that was not finite: all that it is part of is not a number
    vs[own[1][69]] = math.nan
    ks[own[2]] = 0                                               # all scores alike
    vs[own[3][3]] = 3e30 if dtype != torch.float16 else 100.0    # next to what the type holds
    ks[own[4]] = math.nan                                         # no score at all is a number
    got = run_attention(ops, dev, q, pools, b_loc, lens, max_len).cpu()
    assert bool(got[0].isnan().all()) and bool(got[1].isnan().all()) and bool(got[4].isnan().all())
    kd, vd = kp.double() * ks.double()[..., None], vp.double() * vs.double()[..., None]
    want, bound = oracle.attend(q[2:4], kd, vd, own[2:4], PART[dtype])
    oracle.assert_within(got[2:4], want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_q_and_pools_at_other_strides_and_alignments(ops, dev, dtype):
    for d, shift in [(128, 0), (128, 1), (64, 16), (80, 8)]:
        q, pools, b_loc, lens, max_len = batch_of([150, 33, 0], 6, 2, d, dtype, 70)
        (kp, ks), (vp, vs) = pools
        want = run_attention(ops, dev, q, pools, b_loc, lens, max_len) if shift == 0 else None
        n = kp.shape[0]
        both = torch.zeros(n * 2 * 2 * (d + 16) + shift, dtype=torch.int8, device=dev)[shift:].view(n, 2, 2, d + 16)
        both[:, 0, :, :d], both[:, 1, :, :d] = kp.to(dev), vp.to(dev)
        scales = torch.zeros(2, 2, n, device=dev)
        scales[0], scales[1] = ks.t().to(dev), vs.t().to(dev)
        rows_q = torch.randn(3, 10, d, generator=g(71)).to(dtype).to(dev)
        rows_q[:, 2:8] = q.to(dev)
        out = ops.token_decode_attention_int8(rows_q[:, 2:8], both[:, 0, :, :d], scales[0].t(), both[:, 1, :, :d], scales[1].t(), b_loc.to(dev),
                                              lens.to(dev), lens.to(dev), max_len)
        slots = [oracle.slots_of(b_loc, lens, max_len, b) for b in range(3)]
        oracle.assert_within(out, *oracle.attend(q, kp.double() * ks.double()[..., None], vp.double() * vs.double()[..., None], slots, PART[dtype]))
        if want is not None:
            assert_exact(out, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_q_off_any_alignment(ops, dev, dtype):
    q, pools, b_loc, lens, max_len = batch_of([150, 33, 0, 1], 6, 2, 64, dtype, 75)
    want = run_attention(ops, dev, q, pools, b_loc, lens, max_len)
    for view in (lambda x: x[1:1 + q.numel()].view(q.shape), lambda x: x[:4 * 6 * 65].view(4, 6, 65)[..., 1:], lambda x: x[3:3 + 4 * 67 * 6].view(6, 4, 67).transpose(0, 1)[..., :64]):
        moved = view(torch.full((4 * 6 * 70,), 7.0, dtype=dtype, device=dev))
        moved.copy_(q)
        got = ops.token_decode_attention_int8(moved, *[t.to(dev) for pool in pools for t in pool], b_loc.to(dev), lens.to(dev), lens.to(dev), max_len)
        assert_exact(got, want)


def test_no_sequences_and_no_tokens(ops, dev):
    kp, ks = torch.ones(4, 2, 64, dtype=torch.int8, device=dev), torch.ones(4, 2, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.token_decode_attention_int8(torch.zeros(0, 2, 64, device=dev), kp, ks, kp, ks, torch.zeros(0, 5, dtype=torch.int32, device=dev), none, none, 5).shape == (0, 2, 64)
    two = torch.full((2,), 3, dtype=torch.int32, device=dev)
    out = ops.token_decode_attention_int8(torch.ones(2, 4, 64, device=dev), kp, ks, kp, ks, torch.zeros(2, 5, dtype=torch.int32, device=dev), two, two, 0)
    assert bool((out == 0).all())
    empty = torch.zeros(0, 2, 64, device=dev)
    before = kp.clone()
    ops.dest_index_copy_kv_pair_int8(empty, empty, none, kp, ks, kp.clone(), ks.clone())
    assert_exact(kp, before)


# ------------------------------------------------------------------ as they are used
def test_a_decode_step_written_attended_to_and_read_back(ops, dev):
    """New tokens go into the cache, the batch attends to them with what was there, and the rows come back for a later
    prompt: each step against its definition on what the step before left."""
    heads, kv_heads, d = 8, 2, 128
    q, pools, b_loc, lens, max_len = batch_of([1, 40, 333], heads, kv_heads, d, torch.bfloat16, 80)
    on = [t.to(dev) for pool in pools for t in pool]
    for step in range(3):
        k, v = rows(3, kv_heads, d, torch.bfloat16, 81 + step), rows(3, kv_heads, d, torch.bfloat16, 90 + step)
        dest = b_loc[:, max_len - 1]
        ops.dest_index_copy_kv_pair_int8(k.to(dev), v.to(dev), dest.to(dev), *on)
        pools = [oracle.write(*pools[0], k, dest), oracle.write(*pools[1], v, dest)]
        for have, want in zip(on, [t for pool in pools for t in pool]):
            assert_exact(have, want)
        check_attention(ops, dev, q, [(on[0].cpu(), on[1].cpu()), (on[2].cpu(), on[3].cpu())], b_loc, lens, max_len)
        back = ops.index_select_kv_pair_int8(*on, b_loc[2, max_len - 333:max_len].to(dev), dtype=torch.bfloat16)
        index = b_loc[2, max_len - 333:max_len]
        assert_exact(back[0], oracle.read(*pools[0], index, torch.bfloat16))
        assert_exact(back[1], oracle.read(*pools[1], index, torch.bfloat16))
        b_loc = torch.cat([b_loc[:, 1:max_len], torch.tensor([[340 + step], [350 + step], [360 + step]]).to(b_loc.dtype), b_loc[:, max_len - 1:]], 1)
        lens = (lens + 1).clamp(max=max_len)


def test_recorded_into_a_graph_and_replayed_next_to_eager_calls(ops, dev, pkg):
    heads, kv_heads, d = 8, 2, 128
    q, pools, b_loc, lens, max_len = batch_of([900, 40, 333], heads, kv_heads, d, torch.bfloat16, 100)
    on, qd, ld, nd = [t.to(dev) for pool in pools for t in pool], q.to(dev), b_loc.to(dev), lens.to(dev)
    k, v, dest = rows(3, kv_heads, d, torch.bfloat16, 101).to(dev), rows(3, kv_heads, d, torch.bfloat16, 102).to(dev), ld[:, max_len - 1].contiguous()

    def step():
        ops.dest_index_copy_kv_pair_int8(k, v, dest, *on)
        return ops.token_decode_attention_int8(qd, on[0], on[1], on[2], on[3], ld, nd, nd, max_len), ops.index_select_kv_pair_int8(*on, dest, dtype=torch.bfloat16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(6):
            before = pkg.runtime.cachingStats()["num_device_malloc"]
            warm = ops.WorkspaceScope()
            with warm:
                step()
            side.synchronize()
            warm.close()
            if pkg.runtime.cachingStats()["num_device_malloc"] == before:
                break
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        scope = ops.WorkspaceScope()
        with scope:
            got, back = step()
    for i in range(4):
        k.copy_(rows(3, kv_heads, d, torch.bfloat16, 110 + i))
        qd.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        kept = [got.clone(), back[0].clone(), back[1].clone()]
        want = step()                                            # eager work of the same kind between the replays
        torch.cuda.synchronize()
        for have, w in zip(kept, [want[0], *want[1]]):
            assert_exact(have, w)
    del graph
    scope.close()


@pytest.mark.parametrize("tokens", [1500, 5000])                 # repeated slots found by the workgroups, and in workspace beforehand
def test_repeated_slots_recorded_into_two_graphs(ops, dev, pkg, tokens):
    slots = tokens // 2
    pools = [[t.to(dev) for pool in empty_pools(slots, 2, 64, seed=i) for t in pool] for i in range(2)]
    x = [rows(tokens, 2, 64, torch.bfloat16, 120 + i).to(dev) for i in range(2)]
    dest = [torch.randint(0, slots, (tokens,), generator=g(130 + i)).to(dev) for i in range(2)]
    calls = [lambda i=i: ops.dest_index_copy_kv_pair_int8(x[i], x[i], dest[i], *pools[i]) for i in range(2)]
    with recorded(ops, pkg, calls[0]) as (first, _), recorded(ops, pkg, calls[1]) as (second, _):
        for r in range(4):
            for i in range(2):
                dest[i].copy_(torch.randint(0, slots, (tokens,), generator=g(140 + 2 * r + i)))
            before = [t.clone() for t in pools[0] + pools[1]]
            first.replay()
            second.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in pools[0] + pools[1]]
            for t, old in zip(pools[0] + pools[1], before):
                t.copy_(old)
            for call in calls:
                call()
            torch.cuda.synchronize()
            for have, want in zip(kept, pools[0] + pools[1]):
                assert_exact(have, want)


def test_on_another_stream_with_calls_in_flight_on_the_first(ops, dev):
    cases = [batch_of([1500, 700, 3], 8, 2, 128, torch.bfloat16, 120 + i) for i in range(2)]
    want = [run_attention(ops, dev, *c) for c in cases]
    on = [(q.to(dev), [t.to(dev) for p in pools for t in p], b_loc.to(dev), lens.to(dev), m) for q, pools, b_loc, lens, m in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(5):
        for i, (q, pool, loc, lens, m) in enumerate(on):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.token_decode_attention_int8(q, pool[0], pool[1], pool[2], pool[3], loc, lens, lens, m))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for o in outs:
            assert_exact(o, want[i])


def test_the_results_that_are_not_given_are_made(ops, dev):
    (kp, ks), (vp, vs) = empty_pools(9, 3, 16)
    index = torch.tensor([2, 8, 0, 5])
    args = kp.to(dev), ks.to(dev), vp.to(dev), vs.to(dev), index.to(dev)
    want = {dtype: (oracle.read(kp, ks, index, dtype), oracle.read(vp, vs, index, dtype)) for dtype in TYPES}
    for dtype in TYPES:
        mine = torch.empty(4, 3, 16, dtype=dtype, device=dev)
        for given in (dict(dtype=dtype), dict(out_k=mine), dict(out_v=mine), dict(dtype=dtype, out_v=mine), dict(out_k=mine, out_v=torch.empty_like(mine))):
            got = ops.index_select_kv_pair_int8(*args, **given)
            assert got[0].data_ptr() != got[1].data_ptr()
            assert all(got[i] is given[key] for i, key in enumerate(("out_k", "out_v")) if key in given)
            for have, expected in zip(got, want[dtype]):
                assert_exact(have, expected)
    assert ops.index_select_kv_pair_int8(*args)[0].dtype == torch.get_default_dtype()
