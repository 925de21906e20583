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
