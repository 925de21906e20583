"""Decode attention over the paged pools where its kernels could part from its definition: sums that cancel, lengths no table
holds, scores that are not numbers or far from zero, tensors off any alignment."""
import math

import pytest
import torch

from tests import cache_oracle as oracle
from tests import test_gpu_int8_cache as int8
from tests import test_gpu_shared_prefix as shared
from tests.cache_oracle import HALF_STEP
from tests.parity import assert_exact

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def g(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ weights keep the bits of 32
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 20])
def test_int8_sums_that_cancel(ops, dev, dtype, d):
    """Two tokens with the same key and values 127 s and -127 s', s' next to s: half of 127 (s - s') is left, of which weights cut
    to fewer bits than the scales have would show other bits. Both exponentials are 1 and their sum 2 without rounding, so the
    bound is that of the sum over two tokens, (2 + 8) u of the magnitudes, and the rounding of the result."""
    heads, batch = 32, 16
    s = 1 + torch.rand(batch, heads, generator=g(1))
    scales = torch.stack([s, s * (1 + (torch.rand(batch, heads, generator=g(2)) - 0.5) * 2.0 ** -12)], 1)   # [batch, 2, heads]
    kp = torch.randint(-127, 128, (batch, 1, heads, d), generator=g(3), dtype=torch.int8).expand(batch, 2, heads, d).reshape(-1, heads, d)
    vp = torch.tensor([127, -127], dtype=torch.int8).repeat(batch)[:, None, None].expand(-1, heads, d).contiguous()
    q, ks = torch.randn(batch, heads, d, generator=g(4)).to(dtype), torch.full((2 * batch, heads), 2.0 ** -7)
    loc = torch.arange(2 * batch).view(batch, 2)
    got = int8.run_attention(ops, dev, q, [(kp, ks), (vp, scales.reshape(-1, heads).contiguous())], loc, torch.full((batch,), 2), 2)
    sd = scales.double()
    want, sizes = 127 * (sd[:, 0] - sd[:, 1]) / 2, 127 * (sd[:, 0] + sd[:, 1]) / 2
    bound = 10 * U * sizes
    bound += (want.abs() + bound) * HALF_STEP[dtype] + U * (dtype == torch.float16)
    oracle.assert_within(got, want[..., None].expand(-1, -1, d), bound[..., None].expand(-1, -1, d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("where", ["shared", "own"])
def test_sums_that_cancel_behind_a_prefix(ops, dev, dtype, d, where):
    """Three tokens: one with a weight p < 1 and values v, two of the largest score with values that add up to -p v but for its
    last bits. Scores are one product of few bits, so only its scaling and the exponential round: p is off by (2 + 3) u |score| + 4 u
    and u where it is cut, with |score| < 1 by 10 u; sums over three tokens by (3 + 8) u of the magnitudes."""
    heads, n = 8, 64                                               # a head of a token triple for each of n pools' places
    score = -torch.rand(n, heads, generator=g(11)).bfloat16().double()
    p = torch.exp(score)
    v = (1 + torch.rand(n, heads, generator=g(12))).bfloat16().double()
    first = (-p * v).to(dtype).double()
    second = (-p * v - first).to(dtype).double()
    outs, wants, bounds = [], [], []
    q = torch.zeros(1, heads, d, dtype=dtype)
    q[..., 0] = 1
    for i in range(n):
        kk, vv = torch.zeros(4, heads, d, dtype=dtype), torch.zeros(4, heads, d, dtype=dtype)
        kk[0, :, 0] = (score[i] * math.sqrt(d)).to(dtype)
        for t, x in enumerate((v, first, second)):
            vv[t] = x[i][:, None].to(dtype)
        have = kk[0, :, 0].double() / math.sqrt(d)                 # (sqrt(128) does not end: the score that the key stands for)
        p_i = torch.exp(have)
        prefix, loc = (torch.arange(3), torch.tensor([[3]])) if where == "shared" else (torch.tensor([3]), torch.arange(3)[None])
        kk[3, :, 0] = -30000.0 if dtype == torch.float16 else -3e4   # the other side has no weight
        lens = torch.tensor([loc.shape[1]])
        outs.append(shared.run(ops, dev, q, kk, vv, prefix, loc, lens, loc.shape[1]).cpu()[0])
        total = p_i + 2
        want = (p_i * v[i] + first[i] + second[i]) / total
        sizes = (p_i * v[i] + first[i].abs() + second[i].abs()) / total
        bound = (10 * p_i * v[i] / total + 11 * sizes) * U
        wants.append(want), bounds.append(bound + (want.abs() + bound) * HALF_STEP[dtype] + U * (dtype == torch.float16))
    spread = lambda rows: torch.stack(rows)[..., None].expand(-1, -1, d)
    oracle.assert_within(torch.stack(outs), spread(wants), spread(bounds))


# ------------------------------------------------------------------ lengths
LENGTHS = [(torch.int64, [2 ** 31, 2 ** 32 + 5, 2 ** 40, 2 ** 31 - 1, -2 ** 32 + 7, -2 ** 63, 2 ** 63 - 1, 3]),
           (torch.int32, [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 64, 2 ** 31 - 500, 3])]


def cut(lens, max_len):
    return torch.tensor(lens).clamp(0, max_len)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("index,lens", LENGTHS)
@pytest.mark.parametrize("max_len", [40, 600, 4096])
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 1, 128), (4, 4, 128), (2, 1, 18)])
def test_any_length_is_cut_to_the_table(ops, dev, dtype, index, lens, max_len, heads, kv_heads, d):
    """Every launch of a call has to cut a length to the same: one chunk, several, and more than the small merge takes."""
    batch, slots = len(lens), max_len + 200
    q = torch.randn(batch, heads, d, generator=g(21)).to(dtype).to(dev)
    k, v = [torch.randn(slots, kv_heads, d, generator=g(22 + i)).to(dtype).to(dev) for i in range(2)]
    (kp, ks), (vp, vs) = [[t.to(dev) for t in pool] for pool in int8.empty_pools(slots, kv_heads, d)]
    loc = torch.randint(0, slots, (batch, max_len + 3), generator=g(24)).to(index).to(dev)
    prefix = torch.randperm(slots, generator=g(25))[:130].to(index).to(dev)
    start = (torch.arange(batch) * max_len).to(index).to(dev)
    given, within = torch.tensor(lens).to(index).to(dev), cut(lens, max_len).to(index).to(dev)

    def halves(n):
        scores = torch.zeros(heads, batch * max_len, dtype=torch.float32, device=dev)
        ops.token_attention(q, k, scores, loc, start, n, max_len)
        return torch.cat([scores.flatten(), ops.token_softmax_reducev(scores, v, torch.empty_like(q), loc, start, n, max_len).float().flatten()])

    for call in (lambda n: ops.token_decode_attention(q, k, v, loc, start, n, max_len),
                 lambda n: ops.token_decode_attention_int8(q, kp, ks, vp, vs, loc, start, n, max_len),
                 lambda n: ops.token_decode_attention_shared_prefix(q, k, v, prefix, loc, start, n, max_len),
                 halves):
        assert_exact(call(given), call(within))


# ------------------------------------------------------------------ scores that are not numbers, or far from zero
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 8, 64), (8, 1, 128), (12, 4, 80), (2, 1, 18)])
@pytest.mark.parametrize("prefix_len", [0, 1, 40, 250, 9500])      # no, one, several shares, and more than the own tokens end on
def test_a_key_that_is_not_a_number_is_never_left_out(ops, dev, dtype, heads, kv_heads, d, prefix_len):
    lens = [1, 2, 3, 0, 17]
    q, k, v, prefix, loc, n, max_len = shared.batch_of(prefix_len, lens, heads, kv_heads, d, dtype, 60)
    for b, t in ((0, 0), (1, 0), (1, 1), (2, 1), (4, 0), (4, 16)):     # token t of sequence b
        slot = loc[b, max_len - lens[b] + t]
        kept = k[slot, kv_heads - 1].clone()
        k[slot, kv_heads - 1, 3] = math.nan
        got = shared.run(ops, dev, q, k, v, prefix, loc, n, max_len).cpu()
        hit = torch.zeros(len(lens), heads, d, dtype=torch.bool)
        hit[b, heads - heads // kv_heads:] = True
        assert torch.equal(got.isnan(), hit)
        k[slot, kv_heads - 1] = kept


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 8, 64), (8, 1, 128), (2, 1, 18)])
def test_stored_scores_that_are_not_numbers(ops, dev, dtype, heads, kv_heads, d):
    lens, max_len = torch.tensor([1, 2, 40, 5]), 40
    v = torch.randn(90, kv_heads, d, generator=g(65)).to(dtype).to(dev)
    loc, start = torch.randint(0, 90, (4, max_len), generator=g(66)).to(dev), torch.arange(4) * max_len
    for b, t in ((0, 0), (1, 0), (1, 1), (2, 39), (3, 2)):
        scores = torch.randn(heads, 4 * max_len, generator=g(67))
        scores[heads - 1, b * max_len + t] = math.nan
        out = ops.token_softmax_reducev(scores.to(dev), v, torch.empty(4, heads, d, dtype=dtype, device=dev), loc, start.to(dev), lens.to(dev), max_len).cpu()
        hit = torch.zeros(4, heads, d, dtype=torch.bool)
        hit[b, heads - 1] = True
        assert torch.equal(out.isnan(), hit)


@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 8, 64), (8, 1, 128)])
def test_stored_scores_of_minus_infinity(ops, dev, heads, kv_heads, d):
    """Steps of the walk over fp32 rows in which a caller has masked every token, ahead of any that counts, are passed over,
    whatever the values are."""
    dtype = torch.float32
    max_len, masked = 100, 64
    v = torch.randn(200, kv_heads, d, generator=g(68)).to(dtype)
    loc = torch.randperm(200, generator=g(69))[:max_len].repeat(2, 1)
    scores = torch.randn(heads, 2 * max_len, generator=g(70))
    scores[:, :masked] = -math.inf
    poisoned = v.clone()
    poisoned[loc[0, :masked]] = math.nan
    start, lens = torch.tensor([0, max_len]), torch.tensor([max_len, max_len])
    halves = lambda vv: ops.token_softmax_reducev(scores.to(dev), vv.to(dev), torch.empty(2, heads, d, dtype=dtype, device=dev), loc.to(dev), start.to(dev), lens.to(dev), max_len)[0].cpu()
    got, want = halves(poisoned), halves(v)
    assert bool(want.isfinite().all())
    assert_exact(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 20])
@pytest.mark.parametrize("sign", [1, -1])
def test_int8_scores_far_from_zero(ops, dev, dtype, d, sign):
    """Scores of up to 2^60 with either sign, no two within 2^20 of each other: all of the weight is one key's."""
    batch, heads, n = 24, 3, 100
    q = torch.zeros(batch, heads, d)
    q[..., 5] = sign * (1 + torch.rand(batch, heads, generator=g(71))) * 2.0 ** 14
    q = q.to(dtype)
    slots = batch * n
    kp, vp = torch.zeros(slots, heads, d, dtype=torch.int8), torch.randint(-127, 128, (slots, heads, d), generator=g(72), dtype=torch.int8)
    keys = torch.stack([torch.randperm(120, generator=g(73 + i))[:n] + 7 for i in range(batch)])   # 7 ... 126, each once
    kp[..., 5] = keys.view(-1, 1).to(torch.int8)
    ks = ((1 + torch.rand(batch, 1, heads, generator=g(74))) * 2.0 ** torch.linspace(12, 38, batch)[:, None, None]).expand(batch, n, heads).reshape(slots, heads)
    vs = 0.5 + torch.rand(slots, heads, generator=g(75))
    loc = torch.arange(slots).view(batch, n)
    got = int8.run_attention(ops, dev, q, [(kp, ks.contiguous()), (vp, vs)], loc, torch.full((batch,), n), n)
    winner = loc.gather(1, (keys * sign).argmax(1, keepdim=True))[:, 0]
    want = vp[winner].double() * vs[winner].double()[..., None]
    oracle.assert_within(got, want, want.abs() * (HALF_STEP[dtype] + 8 * U))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 2, 128), (20, 1, 64), (2, 2, 256), (2, 1, 18)])
@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_from_zero_behind_a_prefix(ops, dev, dtype, heads, kv_heads, d, where, sign):
    """All elements of a key alike, so scores are 2^28 and more (2^50 where the type holds that) and either equal or far
    apart: the result is the mean of the values with the best key, on the side that has it."""
    lens = [30, 1, 0, 70] * 4
    _, k, v, prefix, loc, n, max_len = shared.batch_of(300, lens, heads, kv_heads, d, torch.float32, 80)
    top = 2.0 ** 13 if dtype == torch.float16 else 2.0 ** 22
    q = (sign * (1 + torch.rand(len(lens), heads, 1, generator=g(81))).expand(-1, -1, d) * top).to(dtype)
    slots = k.shape[0]
    step = torch.randperm(slots, generator=g(82)) % 100            # a few keys alike, some of them among the best
    key = 1 + step / 128
    better = torch.zeros(slots, dtype=torch.bool)
    better[prefix.long() if where == "shared" else torch.cat([oracle.slots_of(loc, n, max_len, b) for b in range(len(lens))])] = True
    key = torch.where(better, key * 2 if sign > 0 else key / 2, key)
    k = (key[:, None, None] * top).expand(slots, kv_heads, d).to(dtype)
    v = (v.sign() * (0.5 + torch.rand(slots, kv_heads, 1, generator=g(83)))).to(dtype)
    got = shared.run(ops, dev, q, k.contiguous(), v, prefix, loc, n, max_len)
    want = torch.zeros(len(lens), heads, d).double()
    for b, seen in enumerate(shared.own_and_shared(prefix, loc, n, max_len)):
        best = (key[seen] * sign) == (key[seen] * sign).max()
        want[b] = v[seen[best]].double().mean(0).repeat_interleave(heads // kv_heads, 0)
    # (ten weights of one at most: (10 + 8) u of values below 1.5, and the rounding)
    oracle.assert_within(got, want, (want.abs() + 27 * U) * HALF_STEP[dtype] + 27 * U + U * (dtype == torch.float16))


# ------------------------------------------------------------------ alignment
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 8, 128), (8, 1, 128), (4, 2, 80), (2, 2, 256), (2, 1, 18)])
@pytest.mark.parametrize("max_len", [30, 900])
def test_results_off_any_alignment(ops, dev, dtype, heads, kv_heads, d, max_len):
    batch = 3
    q, k, v, prefix, loc, n, _ = [t.to(dev) if hasattr(t, "to") else t for t in shared.batch_of(100, [max_len, 1, 7], heads, kv_heads, d, dtype, 90, spare=0)]
    pools = [t.to(dev) for pool in int8.empty_pools(k.shape[0], kv_heads, d) for t in pool]
    for call in (lambda out: ops.token_decode_attention(q, k, v, loc, n, n, max_len, out=out),
                 lambda out: ops.token_decode_attention_int8(q, *pools, loc, n, n, max_len, out=out),
                 lambda out: ops.token_decode_attention_shared_prefix(q, k, v, prefix, loc, n, n, max_len, out=out)):
        want = call(torch.empty_like(q))
        around = torch.full((q.numel() + 9,), 7.0, dtype=dtype, device=dev)
        call(around[1:1 + q.numel()].view(q.shape))
        assert_exact(around[1:1 + q.numel()].view(q.shape), want)
        assert bool((around[1 + q.numel():] == 7).all()) and float(around[0]) == 7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(6, 2, 64), (8, 8, 128), (4, 2, 256)])
def test_q_off_any_alignment_behind_a_prefix(ops, dev, dtype, heads, kv_heads, d):
    """Bit for bit what an aligned q gives: the shared rows are read for many sequences at a time all the same."""
    q, k, v, prefix, loc, n, max_len = [t.to(dev) if hasattr(t, "to") else t for t in shared.batch_of(700, [33, 0, 200, 1], heads, kv_heads, d, dtype, 95)]
    want = ops.token_decode_attention_shared_prefix(q, k, v, prefix, loc, n, n, max_len)
    for view in (lambda x: x[1:1 + q.numel()].view(q.shape), lambda x: x[:4 * heads * (d + 1)].view(4, heads, d + 1)[..., 1:],
                 lambda x: x[3:3 + 4 * heads * (d + 3)].view(heads, 4, d + 3).transpose(0, 1)[..., :d]):
        moved = view(torch.full((4 * heads * (d + 6),), 7.0, dtype=dtype, device=dev))
        moved.copy_(q)
        assert_exact(ops.token_decode_attention_shared_prefix(moved, k, v, prefix, loc, n, n, max_len), want)
