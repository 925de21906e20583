"""GPU parity of the rotation of new q and k rows on their way into the paged cache, against the definition in 64 bits."""
import math

import pytest
import torch

from tests.cache_graph import recorded
from tests.cache_oracle import HALF_STEP
from tests.paged_batch import g
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def rotated(x, cos, sin, interleaved):
    """x [tokens, heads, d] in 64 bits, cos and sin [tokens, d / 2]; and how far a result may be: two products and a sum in 32 bits
    (3 units of 2^-24 of the sizes, and numbers below 2^-126 may be nothing), one rounding to x's type."""
    d, dtype = x.shape[-1], x.dtype
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :d // 2], x[..., d // 2:])
    put = lambda u, v: torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    want, size = put(a * c - b * s, a * s + b * c), put(a.abs() * c.abs() + b.abs() * s.abs(), a.abs() * s.abs() + b.abs() * c.abs())
    bound = 3 * 2.0 ** -24 * size + 2.0 ** -125
    return want, bound + (want.abs() + bound) * HALF_STEP[dtype] + 2.0 ** -25 * (dtype == torch.float16)


def within(got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape and bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound.clamp_min(1e-300)).max())


def case(tokens, heads, kv_heads, d, dtype, seed, *, table=torch.float32, cols=None, slots=None, rows=50):
    gen = g(seed)
    q, k, v = [torch.randn(tokens, n, d, generator=gen).to(dtype) for n in (heads, kv_heads, kv_heads)]
    angle = torch.rand(rows, cols or d // 2, generator=gen) * 6.3
    cos, sin = angle.cos().to(table), angle.sin().to(table)
    slots = slots or tokens + 5
    pools = [torch.randn(slots, kv_heads, d, generator=gen).to(dtype) for _ in range(2)]
    return q, k, v, cos, sin, torch.randint(0, rows, (tokens,), generator=gen), torch.randperm(slots, generator=gen)[:tokens], pools


def halves(t, d, interleaved):
    return t if t.shape[1] != d else t[:, 0::2] if interleaved else t[:, :d // 2]


def check(ops, dev, q, k, v, cos, sin, pos, dest, pools, interleaved, index=torch.int32, by_position=True):
    d, on = k.shape[-1], [p.clone().to(dev) for p in pools]
    got = ops.rotary_dest_index_copy_kv_pair(None if q is None else q.to(dev), k.to(dev), v.to(dev), cos.to(dev), sin.to(dev), dest.to(index).to(dev), *on,
                                             positions=pos.to(index).to(dev) if by_position else None, interleaved=interleaved)
    tokens, slots = k.shape[0], pools[0].shape[0]
    row = pos if by_position else torch.arange(tokens) % cos.shape[0]
    inside = ((row >= 0) & (row < cos.shape[0]))[:, None]
    c, s = [torch.where(inside, halves(t, d, interleaved)[torch.where(inside[:, 0], row, 0)].double(), 0.0) for t in (cos, sin)]
    if q is not None:
        within(got, *rotated(q, c, s, interleaved))
    else:
        assert got is None
    at = torch.where(dest < 0, dest + slots, dest)
    kept = (at >= 0) & (at < slots)
    want, bound = rotated(k, c, s, interleaved)
    within(on[0].cpu()[at[kept]], want[kept], bound[kept])
    assert_exact(on[1].cpu()[at[kept]], v[kept])
    others = torch.ones(slots, dtype=torch.bool)
    others[at[kept]] = False
    for a, b in zip(on, pools):
        assert_exact(a.cpu()[others], b[others])                    # no other slot is touched
    return got, on


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 32, 128), (32, 8, 128), (8, 8, 64), (4, 1, 80), (3, 1, 2), (5, 5, 6), (1, 1, 256), (2, 2, 96), (71, 1, 64), (7, 3, 20), (2, 1, 1024)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_of_any_size(ops, dev, dtype, heads, kv_heads, d, interleaved):
    for tokens in (1, 3, 64, 133):
        for by_position in (True, False):
            x = case(tokens, heads, kv_heads, d, dtype, 10 + tokens, rows=50 if by_position else (tokens if tokens != 64 else 16))
            check(ops, dev, *x, interleaved, torch.int64 if tokens == 3 else torch.int32, by_position)


@pytest.mark.parametrize("dtype,table", [(t, u) for t in TYPES for u in (t, torch.float32)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_tables_of_both_types_and_widths(ops, dev, dtype, table, interleaved, d):
    for cols in (d // 2, d):
        check(ops, dev, *case(37, 8, 2, d, dtype, 30, table=table, cols=cols), interleaved)
        x = list(case(40, 8, 2, d, dtype, 31, table=table, cols=cols, rows=20))
        x[3], x[4] = x[3].t().contiguous().t(), x[4].t().contiguous().t()      # columns first
        check(ops, dev, *x, interleaved, torch.int64, False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_destinations_and_positions_outside(ops, dev, dtype, interleaved):
    for d in (128, 20):
        q, k, v, cos, sin, pos, dest, pools = case(40, 8, 2, d, dtype, 40, slots=60)
        dest = dest - torch.where(torch.arange(40) % 3 == 0, 60, 0)             # some from the end
        dest[5], dest[11], dest[20] = 60, -61, 2 ** 31 - 1
        pos[7], pos[8], pos[20] = -1, 50, 2 ** 31 - 1
        check(ops, dev, q, k, v, cos, sin, pos, dest, pools, interleaved)
        dest[20], pos[20], pos[21] = 2 ** 40, -2 ** 35, 2 ** 33
        check(ops, dev, q, k, v, cos, sin, pos, dest, pools, interleaved, torch.int64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_alignments_and_q_in_place(ops, dev, dtype, interleaved):
    for d, shift in ((128, 0), (128, 1), (64, 8), (80, 4)):
        q, k, v, cos, sin, pos, dest, pools = case(33, 6, 2, d, dtype, 50)
        stacked = torch.cat([q, k, v], 1).to(dev)
        slots = pools[0].shape[0]
        both = torch.full((slots * 2 * 2 * (d + 8) + shift,), 5.0, dtype=dtype, device=dev)[shift:].view(slots, 2, 2, d + 8)
        kp, vp = both[:, 0, :, :d], both[:, 1, :, :d]
        back = ops.rotary_dest_index_copy_kv_pair(stacked[:, :6], stacked[:, 6:8], stacked[:, 8:], cos.to(dev), sin.to(dev), dest.to(dev), kp, vp, positions=pos.to(dev),
                                                  interleaved=interleaved, out_q=stacked[:, :6])
        assert back.data_ptr() == stacked.data_ptr()
        c, s = cos[pos].double(), sin[pos].double()
        within(stacked[:, :6], *rotated(q, c, s, interleaved))
        assert_exact(stacked[:, 6:].cpu(), torch.cat([k, v], 1))
        within(kp.cpu()[dest], *rotated(k, c, s, interleaved))
        assert_exact(vp.cpu()[dest], v)
        left = torch.ones(slots, dtype=torch.bool)
        left[dest] = False
        assert bool((both.cpu()[left] == 5).all() & (both[..., d:] == 5).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_without_q_and_without_tokens(ops, dev, dtype):
    x = list(case(20, 4, 2, 64, dtype, 60))
    check(ops, dev, None, *x[1:], True)
    none = torch.zeros(0, 2, 64, dtype=dtype, device=dev)
    pool = torch.ones(4, 2, 64, dtype=dtype, device=dev)
    table, no = torch.zeros(1, 32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.rotary_dest_index_copy_kv_pair(none, none, none, table, table, no, pool, pool).shape == (0, 2, 64)
    assert bool((pool == 1).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_infinities_and_nan_stay_in_their_pairs(ops, dev, dtype, interleaved):
    q, k, v, cos, sin, pos, dest, pools = case(9, 2, 2, 64, dtype, 70)
    for x in (q, k, v):
        x[4, 1, 6], x[5, 0, 3] = math.inf, math.nan
    on = [p.clone().to(dev) for p in pools]
    got = ops.rotary_dest_index_copy_kv_pair(q.to(dev), k.to(dev), v.to(dev), cos.to(dev), sin.to(dev), dest.to(dev), *on, positions=pos.to(dev), interleaved=interleaved).cpu()
    hit = torch.zeros(9, 2, 64, dtype=torch.bool)
    for t, h, e in ((4, 1, 6), (5, 0, 3)):
        hit[t, h, [e, e ^ 1 if interleaved else e + 32]] = True
    for out, x in ((got, q), (on[0].cpu()[dest], k)):
        assert torch.equal(~out.isfinite(), hit)
        want, bound = rotated(torch.where(hit, torch.zeros((), dtype=dtype), x), cos[pos], sin[pos], interleaved)
        within(out[~hit], want[~hit], bound[~hit])
    assert torch.equal(on[1].cpu()[dest].view(torch.int16 if dtype != torch.float32 else torch.int32), v.view(torch.int16 if dtype != torch.float32 else torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_near_the_separate_calls(ops, dev, dtype, interleaved):
    """What the four calls that it stands for give, up to the rounding of one multiply-add."""
    q, k, v, cos, sin, pos, dest, pools = [t.to(dev) if hasattr(t, "to") else [p.to(dev) for p in t] for t in case(300, 32, 8, 128, dtype, 80)]
    on, other = [p.clone() for p in pools], [p.clone() for p in pools]
    got = ops.rotary_dest_index_copy_kv_pair(q, k, v, cos, sin, dest, *on, positions=pos, interleaved=interleaved)
    c, s = cos[pos], sin[pos]
    ops.dest_index_copy_kv_pair(ops.rotary_emb(k, c, s, interleaved=interleaved), v, dest, *other)
    for a, b in ((got, ops.rotary_emb(q, c, s, interleaved=interleaved)), (on[0], other[0]), (on[1], other[1])):
        a, b = a.double(), b.double()
        assert bool(((a - b).abs() <= 2 * HALF_STEP[dtype] * b.abs() + 2.0 ** -20).all())


def test_far_slots_of_a_pool_past_2_to_the_31_elements(ops, dev):
    slots, heads, d = 270000, 32, 256
    k_pool, v_pool = [torch.zeros(slots, heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    q, k, v, cos, sin, pos, _, _ = case(4, 1, heads, d, torch.bfloat16, 90)
    dest = torch.tensor([slots - 1, 0, 262150, -2])
    ops.rotary_dest_index_copy_kv_pair(q.to(dev), k.to(dev), v.to(dev), cos.to(dev), sin.to(dev), dest.to(dev), k_pool, v_pool, positions=pos.to(dev), interleaved=True)
    at = torch.where(dest < 0, dest + slots, dest).to(dev)
    within(k_pool[at], *rotated(k, cos[pos], sin[pos], True))
    assert_exact(v_pool[at].cpu(), v)


@pytest.mark.parametrize("dtype", TYPES)
def test_recorded_into_a_graph(ops, dev, pkg, dtype):
    q, k, v, cos, sin, pos, dest, pools = [t.to(dev) if hasattr(t, "to") else [p.to(dev) for p in t] for t in case(70, 8, 2, 128, dtype, 100)]
    call = lambda: ops.rotary_dest_index_copy_kv_pair(q, k, v, cos, sin, dest, *pools, positions=pos, interleaved=True)
    with recorded(ops, pkg, call) as (graph, out):
        for i in range(4):
            q.mul_(0.5), k.mul_(0.5), v.add_(1)
            pos.copy_((pos + 7) % 50), dest.copy_(dest.roll(1))
            graph.replay()
            torch.cuda.synchronize()
            kept = [out.clone(), pools[0].clone(), pools[1].clone()]
            pools[0].zero_(), pools[1].zero_()
            want = call()
            torch.cuda.synchronize()
            assert_exact(kept[0], want)
            assert_exact(kept[1][dest], pools[0][dest])
            assert_exact(kept[2][dest], pools[1][dest])
