"""Batches of new tokens over a paged pool, which slots each of them sees, and what attention gives them in 64 bits."""
import math

import torch

from tests.cache_oracle import HALF_STEP


def g(seed):
    return torch.Generator().manual_seed(seed)


class Batch:
    """`new[b]` new tokens of each sequence of `lens[b]`; rows of q in a shuffled order of sequences with gaps between them. Table
    places of no token, and those that no new token sees, hold foreign slots."""

    def __init__(self, new, lens, heads, kv_heads, d, dtype, seed, *, index=torch.int32, window=0, sinks=0, spare=3, gap=2, tail=3):
        gen = g(seed)
        self.window, self.sinks, self.new, self.lens, self.dtype = window, sinks, list(new), list(lens), dtype
        n, self.max_len, self.max_new = len(lens), max(max(lens), 1), max(max(new), 1)
        slots = sum(lens) + 9
        self.k, self.v = [torch.randn(slots, kv_heads, d, generator=gen).to(dtype) for _ in range(2)]
        self.b_loc = torch.randint(0, slots, (n, self.max_len + spare), generator=gen).to(index)
        perm, at = torch.randperm(slots, generator=gen), 0
        for b in range(n):
            for j in self.wanted(b):
                self.b_loc[b, self.max_len - lens[b] + j] = int(perm[at])
                at += 1
        self.start, row = [0] * n, 1 if gap else 0
        for b in torch.randperm(n, generator=gen).tolist() if gap else range(n):
            self.start[b] = row
            row += self.new[b] + (b % (gap + 1) if gap else 0)
        self.rows = row + tail
        self.q = torch.randn(self.rows, heads, d, generator=gen).to(dtype)
        self.tables = [torch.tensor(x).to(index) for x in (self.start, self.new, self.lens)]

    def wanted(self, b):
        """Tokens of sequence b that one of its new ones sees."""
        return sorted({j for t in range(self.new[b]) for j in self.sees(self.lens[b] - self.new[b] + t)})

    def sees(self, p):
        return [j for j in range(p + 1) if not self.window or j > p - self.window or j < self.sinks]

    def slots_of_rows(self):
        """For each row of q the slots of the tokens that it sees, in order (none for rows of no sequence), and the rows of sequences."""
        none = torch.zeros(0, dtype=torch.long)
        seen, owned = [none] * self.rows, [False] * self.rows
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            for t in range(n):
                at = [self.max_len - length + j for j in self.sees(length - n + t)]
                seen[self.start[b] + t] = self.b_loc[b, at].long() if at else none
                owned[self.start[b] + t] = True
        return seen, torch.tensor(owned)

    def attend(self, part):
        """The definition in 64 bits for the rows of sequences, how far a result may be from it, and which rows those are. The bound is the one
        of cache_oracle.attend, which has its derivation, for all rows of a sequence at once."""
        u = 2.0 ** -24
        heads, d = self.q.shape[1:]
        group = heads // self.k.shape[1]
        want, bound = [torch.zeros(self.q.shape).double() for _ in range(2)]
        owned = torch.zeros(self.rows, dtype=torch.bool)
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            rows = slice(self.start[b], self.start[b] + n)
            owned[rows] = True
            j, p = torch.arange(length), torch.arange(length - n, length)[:, None]
            slots = self.b_loc[b, self.max_len - length:self.max_len].long()
            inside = (slots >= 0) & (slots < self.k.shape[0])
            sees = (j <= p) & inside
            if self.window:
                sees &= (j > p - self.window) | (j < self.sinks)
            any_sees = sees.any(0)[:, None, None]
            if not bool(any_sees.any()):
                continue
            kk, vv = [torch.where(any_sees, x[torch.where(inside, slots, 0)], torch.zeros((), dtype=x.dtype)).double().movedim(1, 0).repeat_interleave(group, 0) for x in (self.k, self.v)]
            qq = self.q[rows].double().movedim(1, 0)
            scores = (qq @ kk.transpose(1, 2) / math.sqrt(d)).masked_fill(~sees, -math.inf)
            p = torch.softmax(scores, -1).masked_fill(~sees.any(-1, keepdim=True), 0)
            sizes = (qq.abs() @ kk.abs().transpose(1, 2) / math.sqrt(d)).masked_fill(~sees, 0).amax(-1, keepdim=True)
            e = (d + 4) * u * sizes + 3 * u * scores.abs().masked_fill(~sees, 0).amax(-1, keepdim=True) + 4 * u + part
            all_of_v = sees.double() @ vv.abs()
            bound[rows] = ((2.1 * e + (sees.sum(-1, keepdim=True) + 8) * u) * (p @ vv.abs()) + 2.0 ** -126 * (1 + all_of_v)).movedim(0, 1)
            if self.dtype == torch.float16:
                # fp16 has no numbers below 2^-24: a probability is taken times 2^7 against a maximum that is at most 2^8 too low, so that one of
                # at least 1 is among the sum's, and each loses at most 2^-25 / 2^7 of it besides
                bound[rows] += (2.1 * 2.0 ** -32 * all_of_v).movedim(0, 1)
            want[rows] = (p @ vv).movedim(0, 1)
        return want, bound + (want.abs() + bound) * HALF_STEP[self.dtype] + 2.0 ** -24 * (self.dtype == torch.float16), owned

    def to(self, dev):
        return (self.q.to(dev), self.k.to(dev), self.v.to(dev), self.b_loc.to(dev), *[t.to(dev) for t in self.tables], self.max_new, self.max_len)

    def run(self, ops, dev, **more):
        return ops.paged_context_attention(*self.to(dev), window=self.window, sinks=self.sinks, **more)
