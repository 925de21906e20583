"""Plain definitions, in 64 bits, of the int8 KV cache and of decode attention over any list of rows, and how far a kernel's
attention may be from them."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # relative, round to nearest


def quantise(x):
    """(int8 rows, float32 scales) of rows [..., d]."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    most = torch.where(finite, x.abs().amax(-1), torch.zeros(()).double())
    # (rounding the 64-bit quotient to 32 bits rounds once: a quotient m / 127 of a 24-bit m is never within 2^-32 of a midpoint)
    scale = (most / 127).float()
    q = torch.where(scale[..., None] > 0, x / scale.double()[..., None], torch.zeros(()).double())
    q = torch.where(finite[..., None], q, torch.zeros(()).double()).round().clamp(-127, 127)
    return q.to(torch.int8), torch.where(finite, scale, torch.full((), math.nan))


def write(pool, scale, x, dest):
    """The pool and its scales after the rows went in one after another."""
    pool, scale = pool.clone(), scale.clone()
    q, s = quantise(x)
    for i, slot in enumerate(dest.tolist()):
        slot += pool.shape[0] if slot < 0 else 0
        if 0 <= slot < pool.shape[0]:
            pool[slot], scale[slot] = q[i], s[i]
    return pool, scale


def read(pool, scale, index, dtype):
    inside = (index >= 0) & (index < pool.shape[0])
    i = torch.where(inside, index, 0).long()
    rows = (pool[i].float() * scale[i][..., None]).to(dtype)
    return torch.where(inside[:, None, None], rows, torch.zeros((), dtype=dtype))


def slots_of(b_loc, lens, max_len, b):
    """The slots of sequence b's tokens: the right end of the first max_len columns of its row."""
    n = min(max(int(lens[b]), 0), max_len)
    return b_loc[b, max_len - n:max_len].long()


def attend(q, k, v, slots_of_batch, part):
    """softmax(q . k / sqrt(d)) . v over each sequence's slots (those outside the pool are skipped; without any the result
    is 0), k and v [slots, kv_heads, d] in 64 bits; and the error that each element may have.

    The bound, with u = 2^-24: a score is a sum of d products in some order in 32 bits, off by at most
    (d + 4) u S with S = sum |q k| / sqrt(d), and its difference to the maximum is rounded again, 3 u max |score|; the
    exponential is good to 4 u; a probability is cut to a number of fewer bits, off by at most `part` relative to it. So each
    weight is off by a factor of at most 1 + e with e the sum of these (a little more than twice it, as the sum below the
    fraction line is off alike), the sums over n tokens add (n + 8) u of the sum of magnitudes, and the result is rounded once to q's type. Weights, relative to the largest, and results below
    2^-126 have fewer bits in 32 or may be nothing at all: off by at most 2^-126 absolutely, the first times |v|."""
    u = 2.0 ** -24
    batch, heads, d = q.shape
    want, bound = torch.zeros(batch, heads, d).double(), torch.zeros(batch, heads, d).double()
    group = heads // k.shape[1]
    for b in range(batch):
        slots = slots_of_batch[b]
        slots = slots[(slots >= 0) & (slots < k.shape[0])]
        if not slots.numel():
            continue
        for h in range(heads):
            kk, vv, qq = k[slots, h // group].double(), v[slots, h // group].double(), q[b, h].double()
            scores = (kk @ qq) / math.sqrt(d)
            p = torch.softmax(scores, 0)
            want[b, h] = p @ vv
            sizes = (kk.abs() @ qq.abs()) / math.sqrt(d)
            e = (d + 4) * u * float(sizes.max()) + 3 * u * float(scores.abs().max()) + 4 * u + part
            bound[b, h] = (2.1 * e + (slots.numel() + 8) * u) * (p @ vv.abs()) + 2.0 ** -126 * (1 + vv.abs().sum(0))
    return want, bound + (want.abs() + bound) * HALF_STEP[q.dtype] + 2.0 ** -24 * (q.dtype == torch.float16)


def assert_within(got, want, bound):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} of {want.numel()} out of tolerance; worst {float(((got - want).abs() / bound.clamp_min(1e-300)).nan_to_num(math.inf).max()):.3g} of it"
